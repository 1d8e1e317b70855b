"""paged_attention against the 64-bit oracle.

Bounds, elementwise, with h half a step of the result's type relative to it (of
a subnormal, eps / 2 of the least normal number: f16 holds results below 2^-14
in steps of 2^-24, so a value there is off by up to 2^-25 however small it is),
D the head dim, n the keys of the row, A = sum_j p_j |v_j| and
Z = max_j sum_d |q_d||k_jd| * scale:
  - a score is an fp32 dot product of exact 16-bit operands (error at most
    (D + 2) 2^-24 Z) times an fp32 scale product (two roundings, 2 * 2^-24 |s|)
    minus the maximum in log2 units (2^-24 times its size, at most 2 Z log2 e):
    e = (D + 8) 2^-24 * Z bounds the error of a score, and 2 e that of log p;
  - exp2 adds 2^-22, the join of the parts as much again;
  - a probability, times 2^12 (chunks of prompts; few rows: 2^15) and its block's
    value scale over the largest one, is rounded to f16: 2^-11 of it, or below
    f16's normal numbers (2^-14) half a step of 2^-24, which is 2^-37 of a key of
    the largest value; n keys: n 2^-37 of it, after the division by a sum of at
    least 1;
  - the sums add n 2^-24 of A.
So |out - exact| <= h |exact| + A (2 e + 2^-21 + 2^-11 + 2 n 2^-24) + n 2^-37 max|v|,
|lse - exact| <= 2 e + 2^-21 + n 2^-24 + 4 * 2^-24 |lse|.
"""

import math
import random

import pytest
import torch

from kernelforge_amd.flash_attention_jvp import PagedKVCache, flash_attention, paged_attention
from oracle import paged as orc

pytestmark = pytest.mark.gpu
DEV = "cuda"
E4M3, INT8 = torch.float8_e4m3fn, torch.int8


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def make_cache(blocks, heads, T, D, code, seed=0, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    if code == INT8:
        key, value = (torch.randint(-128, 128, (blocks, heads, T, D), generator=g).to(INT8) for _ in range(2))
        unit = 1 / 64
    else:
        key, value = ((torch.randn(blocks, heads, T, D, generator=g) * 60).clamp(-448, 448).to(E4M3) for _ in range(2))
        unit = 1 / 60
    value = value.view(torch.uint8).reshape(blocks, heads, T // 16, 16, D).transpose(-1, -2).contiguous().view(code)
    # Any positive scale, not only the powers of two that the writes leave.
    scales = [unit * torch.exp(spread * torch.randn(blocks, heads, generator=g)) for _ in range(2)]
    scales[0] = scales[0].clamp(max=3 * unit)
    return PagedKVCache(*(t.to(DEV) for t in (key, value, *scales)))


def bounds(want, out_dtype, cache, D, n):
    out, lse, spread, slack = want
    half, least = torch.finfo(out_dtype).eps / 2, torch.finfo(out_dtype).tiny
    e = (D + 8) * 2.0 ** -24 * slack
    top = float((orc.LARGEST[cache[0].dtype] + 1) * cache[3].abs().nan_to_num(0).max())
    rel = 2 * e.T[..., None] + 2.0 ** -21 + 2.0 ** -11 + 2 * n * 2.0 ** -24
    return half * out.abs().clamp(min=least) + spread * rel + n * 2.0 ** -37 * top, 2 * e + 2.0 ** -21 + n * 2.0 ** -24 + 2.0 ** -22 * lse.abs()


def compare(got, want, limits):
    for have, expect, limit in zip(got, want, limits):
        # Past the largest number of the type (65504 in f16) the rounded result is an infinity.
        most = torch.finfo(have.dtype).max
        over = (expect.abs() - limit > most * (1 + torch.finfo(have.dtype).eps)) & torch.isfinite(expect)
        expect = torch.where(over, expect.sign() * math.inf, expect)
        near = torch.isfinite(expect) & (expect.abs() + limit >= most)  # either is right there
        have = torch.where(near, expect, have.cpu().double())
        assert torch.equal(have.isnan(), expect.isnan())
        assert torch.equal(have.isinf(), expect.isinf())
        fine = torch.isfinite(expect)
        off = (have - expect).abs()[fine] - limit[fine]
        assert off.numel() == 0 or float(off.max()) <= 0, f"{float(off.max()):.3g} past the bound"


def check(q, cache, tables, context, starts, scale=None, causal=True, **kw):
    want = orc.attention(q, cache, tables, context, starts, scale=scale, causal=causal)
    got = paged_attention(q, cache, ints(tables), ints(context), None if starts is None else ints(starts),
                          softmax_scale=scale, causal=causal, return_lse=True, **kw)
    compare(got, want, bounds(want, q.dtype, cache, q.shape[2], max([1, *context])))
    again = paged_attention(q, cache, ints(tables), ints(context), None if starts is None else ints(starts),
                            softmax_scale=scale, causal=causal, return_lse=True, **kw)
    for a, b in zip(got, again):
        assert torch.equal(a.nan_to_num(nan=7.0), b.nan_to_num(nan=7.0))
    return got


def layout(context, T, blocks, rng, width=None):
    """A table of distinct random blocks for each request; -1 behind it."""
    need = [-(-max(c, 0) // T) for c in context]
    ids = rng.sample(range(blocks), sum(need))
    width = width or max([1, *need])
    return [[ids.pop() if j < n else -1 for j in range(width)] for n in need]


def queries(tokens, heads, D, dtype, seed=2):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(tokens, heads, D, generator=g).to(dtype).to(DEV)


SHAPES = [(16, 8, 2, 128), (16, 4, 4, 64), (32, 16, 1, 256), (64, 6, 2, 80), (128, 12, 4, 96), (16, 3, 1, 16),
          (32, 5, 5, 192), (64, 40, 2, 32), (16, 8, 8, 112)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("code", [E4M3, INT8])
@pytest.mark.parametrize("T,Hq,Hkv,D", SHAPES)
def test_decode(T, Hq, Hkv, D, code, dtype):
    """One token a request; contexts of one key, of part and whole of a block and
    of a 64-key tile, an empty one."""
    rng = random.Random(D)
    context = [1, 0, T - 1, T, T + 1, 63, 64, 65, 700]
    cache = make_cache(80, Hkv, T, D, code)
    tables = layout(context, T, 80, rng)
    check(queries(len(context), Hq, D, dtype), cache, tables, context, None)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype,code", [(torch.bfloat16, E4M3), (torch.float16, INT8), (torch.bfloat16, INT8),
                                        (torch.float16, E4M3)])
@pytest.mark.parametrize("T,Hq,Hkv,D", SHAPES)
def test_ragged(T, Hq, Hkv, D, dtype, code, causal):
    """Requests of none, one, a few and many new tokens in one call: more than their
    context (rows that see nothing), all of it, a part."""
    rng = random.Random(D + causal)
    count = [1, 0, 5, 17, 3, 90, 2]
    context = [40, 9, 2, 17, 300, 90, 0]
    starts = [0]
    for n in count:
        starts.append(starts[-1] + n)
    cache = make_cache(60, Hkv, T, D, code)
    tables = layout(context, T, 60, rng)
    q = queries(starts[-1], Hq, D, dtype)
    out, lse = check(q, cache, tables, context, starts, causal=causal, max_query_len=90)
    if causal:  # the first three of five tokens over two keys see none
        assert not out[1:4].any() and lse[:, 1:4].isposinf().all()
    assert not out[-2:].any() and lse[:, -2:].isposinf().all()


@pytest.mark.parametrize("code,dtype", [(E4M3, torch.bfloat16), (INT8, torch.float16)])
@pytest.mark.parametrize("T,Hq,Hkv,D", [(16, 8, 2, 128), (64, 4, 4, 64), (32, 8, 1, 256), (128, 6, 2, 80), (16, 3, 1, 16),
                                        (32, 7, 7, 208)])
def test_prompts(T, Hq, Hkv, D, code, dtype):
    """Chunks of prompts over contexts long enough to be split, beside a decoding
    request and one at the border of the kernels (64 and 65 rows of a key head):
    several tiles of rows, tiles that end inside a block, rows of two queries."""
    rng = random.Random(D)
    group = Hq // Hkv
    count = [1, 64 // group, 64 // group + 1, 150, 33]
    context = [1200, 700, 1030, 1800, 33]
    starts = [0]
    for n in count:
        starts.append(starts[-1] + n)
    cache = make_cache(400, Hkv, T, D, code)
    tables = layout(context, T, 400, rng)
    q = queries(starts[-1], Hq, D, dtype)
    check(q, cache, tables, context, starts, max_query_len=150)
    check(q, cache, tables, context, starts, causal=False, max_context_len=100)


def test_prompt_scores_that_grow():
    """Scores that rise past the rows' references again and again, and value scales
    that do."""
    T, D, c, n = 16, 64, 800, 60
    cache = make_cache(50, 1, T, D, INT8, spread=0.0)
    order = list(range(50))
    cache.key_scale[:, 0] = torch.linspace(0.001, 0.2, 50).to(DEV)
    cache.value_scale[:, 0] = 2.0 ** torch.linspace(-30, 3, 50).to(DEV)
    check(queries(n, 4, D, torch.bfloat16), cache, [order], [c], [0, n])
    check(queries(n, 4, D, torch.float16), cache, [order[::-1]], [c], [0, n], scale=0.5)


@pytest.mark.parametrize("max_context_len", [0, 64, 700, 5000, None])
def test_every_split_count(max_context_len):
    """The bound on the contexts only guides the split: a wrong one costs time."""
    rng = random.Random(1)
    context = [5000, 3, 700]
    cache = make_cache(400, 2, 16, 128, E4M3)
    tables = layout(context, 16, 400, rng)
    q = queries(3, 8, 128, torch.bfloat16)
    check(q, cache, tables, context, None, max_context_len=max_context_len)
    q = queries(9, 8, 128, torch.float16)
    check(q, cache, tables, context, [0, 4, 5, 9], max_context_len=max_context_len, max_query_len=4)


@pytest.mark.parametrize("code", [E4M3, INT8])
def test_scales_far_apart(code):
    """Value scales that span 2^60, keys whose scores grow along the row, a block of
    the least scale (all zeros): no term is lost that the result shows."""
    rng = random.Random(2)
    context, T = [900], 16
    cache = make_cache(57, 1, T, 64, code)
    tables = layout(context, T, 57, rng)
    order = torch.tensor(tables[0])
    cache.value_scale[order] = (2.0 ** torch.linspace(-40, 20, 57))[:, None].to(DEV)
    cache.value_scale[order[3]] = 2.0 ** -126
    check(queries(1, 4, 64, torch.bfloat16), cache, tables, context, None, scale=0.01)
    cache.value_scale[order] = (2.0 ** torch.linspace(20, -40, 57))[:, None].to(DEV)
    check(queries(1, 4, 64, torch.float16) * 0.01, cache, tables, context, None, scale=0.01)
    cache.value_scale[:] = 2.0 ** -126
    got = paged_attention(queries(1, 4, 64, torch.bfloat16), cache, ints(tables), ints(context))
    assert got.isfinite().all()


def test_what_lies_behind_the_context_is_not_looked_at():
    """NaN codes, NaN and infinite scales, blocks that do not exist behind the last
    key; and causal rows are not touched by later keys' blocks."""
    rng = random.Random(3)
    T, D, context, starts = 16, 64, [37, 70], [0, 6, 26]
    cache = make_cache(12, 2, T, D, E4M3)
    tables = layout(context, T, 12, rng, width=9)
    q = queries(26, 4, D, torch.bfloat16)
    want = check(q, cache, tables, context, starts, max_query_len=20)
    raw = [t.view(torch.uint8) for t in cache[:2]]
    for row, c in zip(tables, context):
        last, rest = row[c // T], c % T
        raw[0][last, :, rest:] = 0x7f
        raw[1][last, :, :, :, rest:] = 0xff
    used = {i for row in tables for i in row if i >= 0}
    spare = min(set(range(12)) - used)
    cache.key_scale[spare], cache.value_scale[spare] = math.nan, math.inf
    for row, c in zip(tables, context):
        row[-(-c // T):] = [spare, 2 ** 31 - 1, -2 ** 31, 12][:len(row) - -(-c // T)] + [-1] * max(0, len(row) - -(-c // T) - 4)
    got = paged_attention(q, cache, ints(tables), ints(context), ints(starts), return_lse=True)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("bad", [-1, 12, 2 ** 31 - 1, -2 ** 31])
def test_bad_pages_give_nan_to_the_rows_that_see_them(bad):
    T, D, context, starts = 16, 64, [70, 70], [0, 30, 60]
    rng = random.Random(4)
    cache = make_cache(12, 2, T, D, INT8)
    tables = layout(context, T, 12, rng)
    q = queries(60, 4, D, torch.bfloat16)
    tables[0][3] = bad  # keys 48 to 63: seen by the queries at 48 and behind, tokens 8 ..
    out, lse = check(q, cache, tables, context, starts)
    assert out[:8].isfinite().all() and out[8:30].isnan().all() and out[30:].isfinite().all()
    # A table that is too narrow for its context.
    out = paged_attention(q, cache, ints([t[:3] for t in tables]), ints(context), ints(starts))
    assert out[:8].isfinite().all() and out[8:30].isnan().all()
    # One token, its last key's block missing.
    tables[0][3], tables[0][4] = tables[1][3], bad
    out = paged_attention(q[:2], cache, ints(tables), ints(context))
    assert out[0].isnan().all() and out[1].isfinite().all()


def test_poisoned_blocks():
    """A scale of NaN (of infinity, for values) reaches the rows that see its block
    and no others."""
    T, D, context, starts = 16, 64, [64], [0, 40]
    cache = make_cache(4, 2, T, D, E4M3)
    q = queries(40, 4, D, torch.bfloat16)
    for which, poison in ((2, math.nan), (3, math.nan), (3, math.inf)):
        parts = [t.clone() for t in cache]
        parts[which][2, 1] = poison  # keys 32 to 47 of the second head: tokens 8 and behind
        out = paged_attention(q, parts, ints([[0, 1, 2, 3]]), ints(context), ints(starts))
        assert out[:, :2].isfinite().all() and out[:8].isfinite().all()
        assert out[8:, 2:].isnan().all()


def test_lengths_that_lie():
    """Lengths past the table, negative ones, starts that run backwards or past the
    tokens, a max_query_len that does not hold: NaN or nothing, never a fault."""
    T, D = 16, 64
    cache = make_cache(12, 2, T, D, E4M3)
    tables = ints([[0, 1, 2], [3, 4, 5]])
    q = queries(10, 4, D, torch.float16)
    out = paged_attention(q[:2], cache, tables, ints([2 ** 31 - 1, 48]))
    assert out[0].isnan().all() and out[1].isfinite().all()
    out = paged_attention(q[:2], cache, tables, ints([-2 ** 31, -1]))
    assert not out.any()
    out = paged_attention(q, cache, tables, ints([40, 40]), ints([0, 7, 10]), max_query_len=3)
    assert out[3:7].isnan().all() and out[:3].isfinite().all() and out[7:].isfinite().all()
    for starts in ([5, 2, 9], [0, 2 ** 31 - 1, 3], [-4, -2, -1], [10, 10, 10]):
        paged_attention(q, cache, tables, ints([40, 40]), ints(starts))
    torch.cuda.synchronize()


@pytest.mark.parametrize("few", [True, False])
def test_rows_behind_the_last_request(few):
    T, D = 16, 64
    cache = make_cache(12, 2, T, D, E4M3)
    n = 3 if few else 200
    tables = ints([[0, 1, 2], [3, 4, 5]])
    q = queries(n + 50, 4, D, torch.bfloat16)
    starts = ints([0, 2, n])
    kw = dict(max_query_len=n, return_lse=True)
    out, lse = paged_attention(q, cache, tables, ints([40, 48]), starts, **kw)
    assert not out[n:].any() and lse[:, n:].isposinf().all()
    mine = torch.full_like(q, 3.0)
    got, lse2 = paged_attention(q, cache, tables, ints([40, 48]), starts, out=mine, **kw)
    assert got.data_ptr() == mine.data_ptr() and (got[n:] == 3.0).all()
    assert torch.equal(got[:n], out[:n]) and torch.equal(lse, lse2)


def test_queries_of_any_layout():
    T, D = 16, 64
    cache = make_cache(12, 2, T, D, INT8)
    tables, context = ints([[0, 1, 2], [3, 4, 5]]), ints([33, 48])
    q = queries(2, 4, D, torch.bfloat16)
    want = paged_attention(q, cache, tables, context)
    packed = torch.randn(2, 8, D, device=DEV).to(q.dtype)
    packed[:, 2:6] = q
    for same in (packed[:, 2:6], q.transpose(0, 1).contiguous().transpose(0, 1), q.transpose(1, 2).contiguous().transpose(1, 2),
                 torch.cat([q, q], -1)[..., :D], torch.cat([q.flatten()[:1], q.flatten()])[1:].view(q.shape)):
        assert torch.equal(paged_attention(same, cache, tables, context), want)
    # A block may stand in many tables, and twice in one.
    shared = ints([[3, 4, 5], [3, 4, 5]])
    twice = paged_attention(q[1:].expand(2, -1, -1), cache, shared, ints([48, 48]))
    assert torch.equal(twice[0], want[1]) and torch.equal(twice[1], want[1])


def test_against_flash_attention():
    """The dense operator on the elements the cache stands for."""
    T, D, c, n = 32, 128, 200, 7
    cache = make_cache(7, 2, T, D, INT8, spread=0.0)
    cache.key_scale[:], cache.value_scale[:] = 1 / 64, 1 / 64  # elements are exact in bf16
    k = (cache.key.float() / 64).transpose(1, 2).reshape(1, 7 * T, 2, D)[:, :c].to(torch.bfloat16)
    v = (orc.tokens_of(cache.value.float()) / 64).transpose(1, 2).reshape(1, 7 * T, 2, D)[:, :c].to(torch.bfloat16)
    q = queries(n, 8, D, torch.bfloat16)
    for causal in (True, False):
        dense = flash_attention(q[None], k, v, causal=causal)[0]
        mine = paged_attention(q, cache, ints([list(range(7))]), ints([c]), ints([0, n]), causal=causal)
        # two bf16 results (half a step each) and flash_attention's bf16 probabilities (2^-8 of |v| <= 2)
        torch.testing.assert_close(mine.float(), dense.float(), rtol=2.0 ** -7, atol=2.0 ** -7 * 2)


@pytest.mark.parametrize("code,dtype", [(E4M3, torch.float16), (INT8, torch.bfloat16)])
@pytest.mark.parametrize("T,Hq,Hkv,D", [(16, 8, 2, 128), (64, 4, 4, 64), (32, 8, 1, 256), (128, 6, 2, 96), (16, 3, 1, 16)])
def test_rows_around_the_kernels_border(T, Hq, Hkv, D, code, dtype):
    """Requests of just up to 128 rows of a key head and just past them, in one call
    and alone, cut and whole."""
    rng = random.Random(D + 1)
    group = Hq // Hkv
    count = [128 // group, 128 // group + 1, 1, 128 // group - 1]
    context = [900, 1100, 1500, 90]
    starts = [0]
    for n in count:
        starts.append(starts[-1] + n)
    cache = make_cache(260, Hkv, T, D, code)
    tables = layout(context, T, 260, rng)
    q = queries(starts[-1], Hq, D, dtype)
    check(q, cache, tables, context, starts, max_query_len=max(count))
    check(q, cache, tables, context, starts, max_query_len=max(count), max_context_len=0)
    for b in (0, 1):
        check(q[starts[b]:starts[b + 1]], cache, tables[b:b + 1], context[b:b + 1], [0, count[b]], causal=False)


@pytest.mark.parametrize("B,Hkv", [(700, 2), (4200, 8)])
def test_large_batches(B, Hkv):
    """Several requests for each thread of the sums, more units than a workgroup
    lists at a time, a search over many requests: the requests of a call of their
    own, whole and cut, with and without starts, some of them empty or prompts."""
    T, D = 16, 16
    rng = random.Random(B)
    cache = make_cache(64, Hkv, T, D, INT8, spread=0.0)
    context = [rng.choice([0, 1, 16, 17, 40]) for _ in range(B)]
    table = ints([[rng.randrange(64) for _ in range(3)] for _ in range(B)])
    q = queries(B, 2 * Hkv, D, torch.float16)
    some = sorted(rng.sample(range(B), 40)) + [B - 1]
    got = paged_attention(q, cache, table, ints(context), return_lse=True)
    for kw in (dict(), dict(query_starts=ints(range(B + 1)), max_query_len=1)):
        for bound in (0, 10 ** 6):
            same = paged_attention(q, cache, table, ints(context), return_lse=True, max_context_len=bound, **kw)
            assert torch.equal(same[0], got[0]) and torch.equal(same[1], got[1])
    want = orc.attention(q[some], cache, table[some].tolist(), [context[b] for b in some], None)
    compare((got[0][some], got[1][:, some]), want, bounds(want, q.dtype, cache, D, 40))
    # Of several tokens each, a few of them many; the ones looked at are called alone.
    count = [rng.choice([0, 1, 1, 2, 3]) for _ in range(B)]
    for b in rng.sample(range(B), 9):
        count[b] = rng.randrange(60, 200)
    starts = [0]
    for n in count:
        starts.append(starts[-1] + n)
    q = queries(starts[-1], 2 * Hkv, D, torch.float16)
    long = [b for b in range(B) if count[b] > 3]
    both = [paged_attention(q, cache, table, ints(context), ints(starts), return_lse=True, max_query_len=200,
                            max_context_len=bound) for bound in (0, 10 ** 6)]
    for b in long + some:
        at = slice(starts[b], starts[b + 1])
        want = orc.attention(q[at], cache, table[b:b + 1].tolist(), context[b:b + 1], [0, count[b]])
        for out, lse in both:
            compare((out[at], lse[:, at]), want, bounds(want, q.dtype, cache, D, 40))


def test_out_may_be_the_queries():
    T, D = 16, 64
    cache = make_cache(200, 2, T, D, INT8)
    context, starts = ints([3000, 60, 80]), ints([0, 1, 2, 152])
    tables = ints([list(range(190)), [190] * 190, [191 + k % 9 for k in range(190)]])
    q = queries(152, 8, D, torch.bfloat16)
    want = paged_attention(q, cache, tables, context, starts)
    assert torch.equal(paged_attention(q, cache, tables, context, starts, out=q), want)


@pytest.mark.parametrize("bad", [-1, 90, 2 ** 31 - 1, -2 ** 31])
@pytest.mark.parametrize("n,context", [(100, 170), (300, 1100)])
def test_bad_pages_of_a_prompt(n, context, bad):
    """Many rows over a missing block, with one workgroup a unit and with several."""
    T, D, at = 16, 64, 5
    rng = random.Random(7)
    cache = make_cache(90, 2, T, D, E4M3)
    tables = layout([context], T, 90, rng)
    tables[0][(context - n) // T + at] = bad
    q = queries(n, 8, D, torch.bfloat16)
    first = ((context - n) // T + at) * T - (context - n)  # the first query that sees the block
    out, lse = check(q, cache, tables, [context], [0, n])
    assert out[:first].isfinite().all() and out[first:].isnan().all()
    out = paged_attention(q, cache, ints([tables[0][:(context - n) // T + at]]), ints([context]), ints([0, n]))
    assert out[:first].isfinite().all() and out[first:].isnan().all()


@pytest.mark.parametrize("T,n,context", [(16, 100, 170), (64, 300, 1111)])
def test_poison_in_a_prompt(T, n, context):
    """Scales and codes that only some rows see, and what lies behind the context."""
    D, blocks = 64, 90
    rng = random.Random(8)
    cache = make_cache(blocks, 2, T, D, E4M3)
    tables = layout([context], T, blocks, rng, width=-(-context // T) + 3)
    q = queries(n, 8, D, torch.bfloat16)
    want = check(q, cache, tables, [context], [0, n])
    at = (context - n) // T + 1
    first = at * T - (context - n)
    for which, poison in ((2, math.nan), (3, math.nan), (3, math.inf)):
        parts = [t.clone() for t in cache]
        parts[which][tables[0][at], 1] = poison
        out = paged_attention(q, parts, ints(tables), ints([context]), ints([0, n]))
        assert out[:first].isfinite().all() and torch.equal(out[:, :4], want[0][:, :4])
        assert out[first:, 4:].isnan().all()
    raw = [t.view(torch.uint8) for t in cache[:2]]
    row, rest = tables[0], context % T
    raw[0][row[context // T], :, rest:] = 0x7f
    for token in range(rest, T):
        raw[1][row[context // T], :, token // 16, :, token % 16] = 0xff
    used = {i for i in row if i >= 0}
    spare = min(set(range(blocks)) - used)
    cache.key_scale[spare], cache.value_scale[spare] = math.nan, math.inf
    row[-3:] = [spare, 2 ** 31 - 1, -2 ** 31]
    for have, expect in zip(paged_attention(q, cache, ints(tables), ints([context]), ints([0, n]), return_lse=True), want):
        assert torch.equal(have, expect)


def test_lengths_that_lie_in_prompts():
    """As in the few-rows kernel: NaN or nothing, and nothing outside the tensors."""
    T, D = 16, 64
    cache = make_cache(12, 2, T, D, E4M3)
    tables = ints([[0, 1, 2], [3, 4, 5], [6, 7, 8]])
    q = queries(400, 4, D, torch.float16)
    starts = ints([0, 150, 300, 400])
    out = paged_attention(q, cache, tables, ints([2 ** 31 - 1, 48, -2 ** 31]), starts)
    assert out[:150].isnan().all() and out[150:300].isfinite().all() and not out[300:].any()
    out = paged_attention(q, cache, tables, ints([40, 40, 40]), starts, max_query_len=120)
    want = paged_attention(q, cache, tables, ints([40, 40, 40]), starts)
    for b, n in ((0, 150), (150, 150), (300, 100)):
        assert torch.equal(out[b:b + min(n, 120)], want[b:b + min(n, 120)]) and out[b + 120:b + n].isnan().all()
    for lie in ([0, 300, 0, 300], [399, 2, 2 ** 31 - 1, 7], [-2 ** 31, 2 ** 31 - 1, -1, 400], [400, 0, 400, 0]):
        paged_attention(q, cache, tables, ints([40, 40, 40]), ints(lie))
    torch.cuda.synchronize()


def test_prompts_on_another_stream_and_captured():
    """A batch that takes both kernels and both joins, in two graphs that are
    replayed in turn on changed inputs, with eager work between."""
    T, D = 16, 128
    cache = make_cache(600, 2, T, D, INT8)
    tables, context, starts = ints([list(range(300)), list(range(300, 600))]), ints([4000, 4500]), ints([0, 1, 201])
    args = (cache, tables, context, starts)
    inputs = [queries(201, 8, D, torch.bfloat16, seed=k) for k in range(3)]
    want = [paged_attention(x, *args) for x in inputs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = paged_attention(inputs[0], *args)
    here = paged_attention(inputs[1], *args)  # at the same time
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want[0]) and torch.equal(here, want[1])
    static, graphs, outs = [inputs[0].clone(), inputs[1].clone()], [], []
    for x in static:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(paged_attention(x, *args))
        graphs.append(graph)
    for k in (0, 2, 1, 2):
        static[0].copy_(inputs[k])
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[k]) and torch.equal(outs[1], want[1])
        assert torch.equal(paged_attention(inputs[2], *args), want[2])


def test_one_head_of_any_stride():
    """A dimension of one may have any stride (a view of [tokens, D])."""
    cache = make_cache(4, 1, 16, 64, INT8)
    tables, context = ints([[0, 1], [2, 3]]), ints([20, 32])
    q = queries(2, 1, 64, torch.bfloat16)
    want = paged_attention(q, cache, tables, context)
    assert torch.equal(paged_attention(q.as_strided((2, 1, 64), (64, 1, 1)), cache, tables, context), want)
    assert torch.equal(paged_attention(q[:1].as_strided((1, 1, 64), (3, 5, 1)), cache, tables[:1], context[:1]), want[:1])


def test_past_32_bits():
    """Blocks whose bytes lie past 2^32 in the caches."""
    T, H, D = 128, 8, 128
    blocks = (1 << 32) // (T * H * D) + 2
    small = make_cache(2, H, T, D, INT8)
    key, value = (torch.zeros((blocks, *t.shape[1:]), dtype=INT8, device=DEV) for t in small[:2])
    scales = [torch.zeros(blocks, H, device=DEV) for _ in range(2)]
    large = PagedKVCache(key, value, *scales)
    for a, b in zip(large, small):
        a[-2:] = b
    q = queries(1, 16, D, torch.bfloat16)
    want = paged_attention(q, small, ints([[1, 0]]), ints([201]))
    assert torch.equal(paged_attention(q, large, ints([[blocks - 1, blocks - 2]]), ints([201])), want)


def test_on_another_stream_and_captured():
    """Calls on a side stream, and a captured call replayed on changed inputs with
    eager work between, two graphs at once."""
    T, D = 16, 128
    cache = make_cache(600, 2, T, D, E4M3)
    tables, context = ints([list(range(300)), list(range(300, 600))]), ints([4000, 4500])
    q, q2 = queries(2, 8, D, torch.bfloat16), queries(2, 8, D, torch.bfloat16, seed=9)
    want, want2 = paged_attention(q, cache, tables, context), paged_attention(q2, cache, tables, context)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = paged_attention(q, cache, tables, context)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    static, graphs, outs = [q.clone(), q.clone()], [], []
    for x in static:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(paged_attention(x, cache, tables, context))
        graphs.append(graph)
    for fresh, expect in ((q, want), (q2, want2), (q, want)):
        static[0].copy_(fresh)
        static[1].copy_(q2)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], expect) and torch.equal(outs[1], want2)
        assert torch.equal(paged_attention(q, cache, tables, context), want)


def test_no_tokens_and_refused_gradients():
    cache = make_cache(2, 2, 16, 64, INT8)
    q = torch.empty(0, 4, 64, dtype=torch.bfloat16, device=DEV)
    out, lse = paged_attention(q, cache, ints([[0]]), ints([3]), ints([0, 0]), return_lse=True)
    assert out.shape == q.shape and lse.shape == (4, 0)
    q = queries(1, 4, 64, torch.bfloat16).requires_grad_()
    with pytest.raises(RuntimeError, match="no backward"):
        paged_attention(q, cache, ints([[0]]), ints([3]))
    with torch.no_grad():
        paged_attention(q, cache, ints([[0]]), ints([3]))
