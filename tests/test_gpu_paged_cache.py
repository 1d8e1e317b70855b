"""Block tables, slots and cache writes on the GPU against the plain oracle.

Both are exact: the tables are whole numbers, and with power-of-two scales every
quotient is exact and rounded once, so codes and scales are the oracle's.
"""

import math
import random

import pytest
import torch

from kernelforge_amd.flash_attention_jvp import PagedKVCache, paged_block_tables_, paged_cache_append_, paged_kv_cache
from oracle import paged as orc

pytestmark = pytest.mark.gpu
DEV = "cuda"
E4M3, INT8 = torch.float8_e4m3fn, torch.int8


def ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEV)


# ---------------------------------------------------------------------------
# Tables.
# ---------------------------------------------------------------------------
def check_tables(tables, context, queries, free, used, total, T, in_place=False):
    want = orc.block_tables(tables, context, queries, free, used, total, T)
    width = len(tables[0])
    dev = ints(tables).reshape(len(tables), width)
    c, u = ints(context), ints([used])
    starts, after, slots, used_out = paged_block_tables_(dev, c, ints(queries), ints(free), u, total_tokens=total,
                                                         block_tokens=T, in_place=in_place)
    got = (dev.tolist(), starts.tolist(), after.tolist(), slots.tolist(), used_out.item())
    assert got == (want[0], *want[1:4], want[4])
    if in_place:
        assert after.data_ptr() == c.data_ptr() and used_out.data_ptr() == u.data_ptr()
    else:
        assert c.tolist() == context and u.item() == used


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("T", [16, 32, 64, 128])
@pytest.mark.parametrize("B", [1, 2, 63, 513, 4096])
def test_tables(B, T, in_place):
    """Every batch size class (more requests than threads, than a scan's wavefront),
    requests of no new tokens, empty ones, block borders; a buffer past the
    tokens; with 513 and more requests several workgroups."""
    rng = random.Random(B + T)
    context = [rng.choice([0, 0, 1, T - 1, T, T + 1, rng.randrange(5 * T)]) for _ in range(B)]
    queries = [rng.choice([0, 1, 1, 2, T, rng.randrange(1, 3 * T if B < 600 else 4)]) for _ in range(B)]
    need = [-(-(c + n) // T) - -(-c // T) for c, n in zip(context, queries)]
    width = max(-(-(c + n) // T) for c, n in zip(context, queries)) + 1
    ids = rng.sample(range(10 ** 6), sum(need) + 7 + B * width)
    free, held = ids[:sum(need) + 7], ids[sum(need) + 7:]
    tables = [[held[b * width + j] if j < -(-c // T) else -5 for j in range(width)] for b, c in enumerate(context)]
    check_tables(tables, context, queries, free, 3, sum(queries) + rng.choice([0, 1, 9]), T, in_place)


@pytest.mark.parametrize("in_place", [False, True])
def test_tables_when_something_is_short(in_place):
    """No block left, a table too narrow, a buffer too short, a count past the
    list or below it, entries that are no block, negative lengths, no tokens."""
    T = 16
    check_tables([[1, -1, -1], [2, -1, -1]], [16, 3], [20, 40], [7, 8], 0, 60, T, in_place)
    check_tables([[1, -1, -1], [2, -1, -1]], [16, 3], [20, 40], [7, 8], 2, 60, T, in_place)
    check_tables([[1], [2]], [10, 3], [20, 40], [7, 8, 9, 10, 11], 1, 70, T, in_place)
    check_tables([[1, -1, -1], [2, -1, -1]], [16, 3], [20, 40], [7, 8, 9, 10], 0, 33, T, in_place)
    check_tables([[1, -1, -1], [2, -1, -1]], [16, 3], [20, 40], [7, 8, 9, 10], 0, 20, T, in_place)
    check_tables([[-3, -1, -1], [2, -1, -1]], [5, -4], [20, 40], [-7, 8, 9, 10], -1, 60, T, in_place)
    check_tables([[1, -1]], [5], [-2], [7], 0, 0, T, in_place)
    check_tables([[]], [0], [3], [], 0, 3, T, in_place)


def test_tables_of_many_workgroups_in_place():
    """The lengths change only after every workgroup has read them."""
    B, T = 300, 16
    context, queries = [5 * b % 90 for b in range(B)], [50 + b % 40 for b in range(B)]
    free = list(range(5000, 5000 + 4000))
    tables = [[1000 + b * 12 + j for j in range(12)] for b in range(B)]
    check_tables(tables, context, queries, free, 0, sum(queries), T, True)


# ---------------------------------------------------------------------------
# Writes.
# ---------------------------------------------------------------------------
def filled(blocks, heads, T, D, dtype, seed=0):
    """A cache of random codes and scales, none of them a NaN."""
    g = torch.Generator().manual_seed(seed)
    if dtype == INT8:
        key, value = (torch.randint(-127, 128, (blocks, heads, T, D), generator=g).to(INT8) for _ in range(2))
    else:
        key, value = ((torch.randn(blocks, heads, T, D, generator=g) * 60).clamp(-448, 448).to(E4M3) for _ in range(2))
    value = value.view(torch.uint8).reshape(blocks, heads, T // 16, 16, D).transpose(-1, -2).contiguous().view(dtype)
    scales = [2.0 ** torch.randint(-12, 2, (blocks, heads), generator=g) for _ in range(2)]
    return PagedKVCache(*(t.to(DEV) for t in (key, value, *scales)))


def check_append(cache, key, value, slots, repeat=True):
    want = orc.append([t.cpu() for t in cache], key.cpu(), value.cpu(), slots)
    got = paged_cache_append_(cache, key, value, ints(slots, torch.int64))
    assert got is cache

    def same():
        for have, expect in zip((cache[0].double(), orc.tokens_of(cache[1].double()), cache[2].double(),
                                 cache[3].double()), want):
            assert torch.equal(have.cpu().nan_to_num(nan=1e30), expect.nan_to_num(nan=1e30))

    same()
    if repeat:  # the same tokens again change nothing
        paged_cache_append_(cache, key, value, ints(slots, torch.int64))
        same()


def tokens(n, heads, D, dtype, seed=1, spread=1.5):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, 2 * heads, D, generator=g) * torch.exp(spread * torch.randn(n, 2 * heads, 1, generator=g))
    x = x.to(dtype).to(DEV)
    return x[:, :heads], x[:, heads:]  # parts of one tensor


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("code", [E4M3, INT8])
@pytest.mark.parametrize("T,D,heads", [(16, 128, 3), (16, 16, 1), (16, 80, 5), (32, 64, 2), (64, 256, 1), (64, 112, 3),
                                       (128, 96, 2), (128, 64, 1), (32, 192, 4), (16, 32, 8)])
def test_append(T, D, heads, code, dtype):
    """Every block size, head-dim class and type: whole blocks, blocks begun in the
    middle (held codes are scaled down), ended early (the rest keeps or becomes
    0), single tokens, skipped slots between requests."""
    cache = filled(12, heads, T, D, code)
    slots = [4 * T + i for i in range(2 * T)]                 # two whole blocks, begun
    slots += [-1, 7 * T + 5, -1]                              # one token, no start
    slots += [2 * T + i for i in range(T - 3, T)] + [9 * T + i for i in range(T // 2)]  # across a border
    slots += [12 * T, 10 * T + 7, 10 * T + 8, 2 ** 40, -2 ** 63, 11 * T]
    key, value = tokens(len(slots), heads, D, dtype)
    check_append(cache, key, value, slots)


@pytest.mark.parametrize("code", [E4M3, INT8])
def test_append_many_runs_in_a_slice(code):
    """Enough tokens that a workgroup takes a block's worth of them, with runs that
    begin anywhere in it, and one that is longer than a block."""
    T, D, heads, blocks = 16, 64, 8, 700
    rng = random.Random(5)
    cache = filled(blocks, heads, T, D, code)
    slots, order = [], rng.sample(range(blocks), blocks - 1)
    while len(order) > 1:
        block, a = order.pop(), rng.randrange(T)
        slots += [block * T + i for i in range(a, rng.randrange(a, T) + 1)]
        if rng.random() < 0.2:
            slots.append(rng.choice([-1, blocks * T]))
    slots += [order.pop() * T + 3] * 40
    key, value = tokens(len(slots), heads, D, torch.bfloat16)
    check_append(cache, key, value, slots)


@pytest.mark.parametrize("T,heads,count", [(16, 32, 150), (32, 8, 300), (32, 32, 700), (64, 8, 300), (64, 32, 500),
                                           (64, 32, 1400), (128, 32, 1400), (128, 32, 2500)])
def test_append_slices_of_every_length(T, heads, count):
    """Workgroups of 2 to 64 tokens: prompts whose runs end anywhere in a slice,
    decoding tokens between them, runs around the 64th slot, padding at the end."""
    D, blocks = 16, 300
    rng = random.Random(count + T)
    cache = filled(blocks, heads, T, D, INT8 if count % 200 else E4M3)
    slots, order = [], rng.sample(range(blocks), blocks)
    while len(slots) < count:
        if rng.random() < 0.6:  # a prompt behind some cached tokens
            at, n = rng.randrange(T), rng.randrange(1, 3 * T)
            while n > 0:
                block, here = order.pop(), min(n, T - at)
                slots += [block * T + at + i for i in range(here)]
                at, n = 0, n - here
        else:
            slots += [order.pop() * T + rng.randrange(T) for _ in range(rng.randrange(1, 6))]
        if rng.random() < 0.2:
            slots += [-1] * rng.randrange(1, 70)
    slots += [-1] * 3
    key, value = tokens(len(slots), heads, D, torch.float16)
    check_append(cache, key, value, slots)


@pytest.mark.parametrize("code", [E4M3, INT8])
def test_append_the_same_slot_twice(code):
    """Of two tokens of a run that name one slot the later is kept, alone."""
    cache = filled(4, 2, 16, 64, code)
    slots = [16 + 3, 16 + 4, 16 + 3, 16 + 3, 2 * 16, 2 * 16]
    key, value = tokens(len(slots), 2, 64, torch.float16)
    key[0] *= 1000  # not kept: it sets no scale
    check_append(cache, key, value, slots)


@pytest.mark.parametrize("code", [E4M3, INT8])
def test_append_token_by_token(code):
    """A decoding loop: the block's scale grows as larger elements arrive."""
    heads, D, T = 2, 64, 32
    cache = paged_kv_cache(3, heads, D, block_tokens=T, dtype=code)
    key, value = tokens(T + 3, heads, D, torch.bfloat16, spread=2.0)
    for t in range(T + 3):
        check_append(cache, key[t:t + 1], value[t:t + 1], [T + t], repeat=False)


@pytest.mark.parametrize("code", [E4M3, INT8])
def test_append_extremes(code):
    """Zeros, the least and the largest of bf16, values on the border of a scale,
    infinities and NaNs (the scale is NaN until the block is begun again)."""
    heads, D, T = 1, 32, 16
    most = orc.LARGEST[code]
    cache = filled(8, heads, T, D, code)
    x = torch.zeros(8, heads, D)
    x[1] = 1e-40
    x[2, :, 0], x[2, :, 1] = 3.3e38, -3.3e38
    x[3, :, 5] = -most * 2.0 ** 3                       # exactly the largest code
    x[4] = torch.linspace(-most, most, D)
    x[5, :, 7], x[6, :, 7], x[7, :, 9] = math.inf, math.nan, -math.inf
    x = x.to(torch.bfloat16).to(DEV)
    check_append(cache, x, x.flip(2).contiguous(), [b * T for b in range(8)])
    assert cache.key_scale[:5].isfinite().all() and cache.key_scale[5:].isnan().all()
    check_append(cache, x[4:5], x[4:5], [5 * T + 1])       # still poisoned
    assert cache.key_scale[5].isnan().all()
    check_append(cache, x[4:5], x[4:5], [5 * T])           # begun again
    assert cache.key_scale[5].isfinite().all()
    check_append(cache, x[5:6], x[4:5], [1 * T + 2])       # a sound block meets an infinity
    assert cache.key_scale[1].isnan().all() and cache.value_scale[1].isfinite().all()


def test_append_rows_of_any_layout():
    """Strides, alignments and orders of the new tokens: copied where need be."""
    heads, D, T = 2, 64, 16
    for make in (lambda x: x, lambda x: x.transpose(0, 1).contiguous().transpose(0, 1),
                 lambda x: x.transpose(1, 2).contiguous().transpose(1, 2),
                 lambda x: torch.cat([x, x], -1)[..., 3:3 + D], lambda x: x.flip(0),
                 lambda x: torch.cat([x.flatten()[:1], x.flatten()])[1:].view(x.shape),
                 lambda x: x[:, :1].expand(-1, heads, -1)):
        cache = filled(3, heads, T, D, E4M3)
        key, value = tokens(7, heads, D, torch.bfloat16)
        check_append(cache, make(key), make(value), [T + 4 + i for i in range(7)])


def test_append_past_32_bits():
    """Blocks whose codes lie past 2^32 bytes."""
    heads, D, T = 8, 128, 128
    blocks = (1 << 32) // (heads * D * T) + 3
    cache = paged_kv_cache(blocks, heads, D, block_tokens=T)
    key, value = tokens(5, heads, D, torch.bfloat16)
    slots = [(blocks - 1) * T + 3 + i for i in range(5)]
    paged_cache_append_(cache, key, value, ints(slots, torch.int64))
    small = paged_kv_cache(1, heads, D, block_tokens=T)
    paged_cache_append_(small, key, value, ints([3 + i for i in range(5)], torch.int64))
    for large, expect in zip(cache, small):
        last = large[-1:]
        assert torch.equal(last.view(torch.uint8) if last.element_size() == 1 else last,
                           expect.view(torch.uint8) if expect.element_size() == 1 else expect)
        # and nowhere else: the block whose address is the last one's modulo 2^32
        assert not large[:4].float().any()


def test_refuses_gradients():
    cache = paged_kv_cache(2, 2, 64)
    key, value = tokens(1, 2, 64, torch.bfloat16)
    key = key.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="no backward"):
        paged_cache_append_(cache, key, value, ints([0], torch.int64))
    with torch.no_grad():
        paged_cache_append_(cache, key, value, ints([0], torch.int64))
