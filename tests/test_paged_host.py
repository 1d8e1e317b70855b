"""The paged cache on the CPU: refusals, where bad pages and lengths lead, and the oracle."""

import ctypes
import math

import pytest
import torch

from kernelforge_amd import _lib
from kernelforge_amd.flash_attention_jvp import (paged_attention, paged_block_tables_, paged_cache_append_,
                                                 paged_kv_cache)
from oracle import fa as ofa
from oracle import paged as orc

i32 = torch.int32


def cache(blocks=4, heads=2, dim=64, T=16, dtype=torch.int8):
    return paged_kv_cache(blocks, heads, dim, block_tokens=T, dtype=dtype, device="cpu")


def ints(*values, dtype=i32):
    return torch.tensor(values, dtype=dtype)


def attend(q=None, kv=None, tables=None, context=None, starts=None, **kw):
    q = torch.zeros(1, 4, 64, dtype=torch.bfloat16) if q is None else q
    return paged_attention(q, kv or cache(), torch.zeros(1, 4, dtype=i32) if tables is None else tables,
                           ints(3) if context is None else context, starts, **kw)


@pytest.mark.parametrize("bad,match", [
    (dict(q=torch.zeros(1, 4, 64)), "bfloat16"),
    (dict(q=torch.zeros(4, 64, dtype=torch.bfloat16)), "tokens, heads"),
    (dict(q=torch.zeros(1, 3, 64, dtype=torch.bfloat16)), "multiple of its heads"),
    (dict(q=torch.zeros(1, 4, 32, dtype=torch.bfloat16)), "head dim"),
    (dict(q=torch.zeros(2, 4, 64, dtype=torch.bfloat16)), "one token of every request"),
    (dict(tables=torch.zeros(1, 4, dtype=torch.int64)), "int32"),
    (dict(tables=torch.zeros(1, 0, dtype=i32)), "neither of them 0"),
    (dict(tables=torch.zeros(1, 8, dtype=i32)[:, ::2]), "contiguous"),
    (dict(context=ints(3, 4)), "context_lens"),
    (dict(context=ints(3, dtype=torch.int64)), "int32"),
    (dict(starts=ints(0, 1, 2)), "query_starts"),
    (dict(softmax_scale=0.0), "positive"),
    (dict(softmax_scale=math.nan), "finite"),
    (dict(starts=ints(0, 1), max_query_len=0), "max_query_len"),
    (dict(max_context_len=-1), "max_context_len"),
    (dict(out=torch.zeros(1, 4, 64, dtype=torch.float16)), "out"),
    (dict(out=torch.zeros(1, 64, 4, dtype=torch.bfloat16).transpose(1, 2)), "out"),
    (dict(kv=cache()[:2] + (torch.zeros(4, 3),) * 2), "scales"),
    (dict(kv=cache()[:2] + (torch.zeros(4, 2, dtype=torch.float16),) * 2), "scales"),
    (dict(kv=(cache()[0], cache(T=32)[1], *cache()[2:])), "value cache"),
    (dict(kv=(cache()[0], cache(dtype=torch.float8_e4m3fn)[1], *cache()[2:])), "value cache"),
    (dict(kv=(cache()[0].float(), *cache()[1:])), "dtype"),
    (dict(kv=(cache()[0][:, :, :, ::2], cache(dim=32)[1], *cache()[2:]), q=torch.zeros(1, 4, 32, dtype=torch.float16)),
     "contiguous"),
    (dict(), "HIP"),  # sound, but on the CPU: refused, never computed
])
def test_attention_refuses(bad, match):
    with pytest.raises(ValueError, match=match):
        attend(**bad)


def append(key=None, value=None, slots=None, kv=None):
    key = torch.zeros(3, 2, 64, dtype=torch.float16) if key is None else key
    return paged_cache_append_(kv or cache(), key, key if value is None else value,
                               ints(0, 1, 2, dtype=torch.int64) if slots is None else slots)


@pytest.mark.parametrize("bad,match", [
    (dict(key=torch.zeros(3, 2, 64)), "bfloat16"),
    (dict(key=torch.zeros(3, 128, dtype=torch.float16)), "tokens, heads"),
    (dict(key=torch.zeros(3, 1, 64, dtype=torch.float16)), "2 heads of 64"),
    (dict(value=torch.zeros(2, 2, 64, dtype=torch.float16)), "value"),
    (dict(value=torch.zeros(3, 2, 64, dtype=torch.bfloat16)), "value"),
    (dict(slots=ints(0, 1, 2)), "int64"),
    (dict(slots=ints(0, 1, dtype=torch.int64)), "slots"),
    (dict(kv=cache()[:3]), "unpack"),
    (dict(), "HIP"),
])
def test_append_refuses(bad, match):
    with pytest.raises(ValueError, match=match):
        append(**bad)


def tables(block_tables=None, context=None, queries=None, free=None, used=None, total=4, T=16):
    return paged_block_tables_(torch.zeros(1, 4, dtype=i32) if block_tables is None else block_tables,
                               ints(3) if context is None else context, ints(4) if queries is None else queries,
                               ints(7) if free is None else free, ints(0) if used is None else used,
                               total_tokens=total, block_tokens=T)


@pytest.mark.parametrize("bad,match", [
    (dict(block_tables=torch.zeros(4, dtype=i32)), "requests, width"),
    (dict(block_tables=torch.zeros(0, 4, dtype=i32)), "hold a request"),
    (dict(context=ints(3, 3)), "context_lens"),
    (dict(queries=ints(3, dtype=torch.int64)), "query_lens"),
    (dict(free=ints(7)[None]), "one dimension"),
    (dict(used=ints(0, 0)), "free_used"),
    (dict(total=-1), "total_tokens"),
    (dict(T=24), "block_tokens"),
    (dict(), "HIP"),
])
def test_tables_refuse(bad, match):
    with pytest.raises(ValueError, match=match):
        tables(**bad)


@pytest.mark.parametrize("args,match", [((0, 2, 64), "positive"), ((4, 0, 64), "positive"), ((4, 2, 72), "multiple of 16"),
                                        ((4, 2, 272), "multiple of 16")])
def test_cache_refuses(args, match):
    with pytest.raises(ValueError, match=match):
        paged_kv_cache(*args, device="cpu")
    with pytest.raises(ValueError, match="block_tokens"):
        paged_kv_cache(4, 2, 64, block_tokens=8, device="cpu")
    with pytest.raises(ValueError, match="dtype"):
        paged_kv_cache(4, 2, 64, dtype=torch.uint8, device="cpu")


def test_c_entries_refuse_before_a_device():
    """Every refusal of the C entries comes before a launch; sound empty calls succeed."""
    lib = _lib.load()
    null = ctypes.c_void_p(0)

    def attn(tokens=4, B=4, blocks=8, width=4, Hq=4, Hkv=2, D=64, T=16, qs=(256, 64), mq=1, mc=64, scale=0.1,
             dtype=_lib.KF_BF16, cdt=_lib.KF_CACHE_INT8, starts=null):
        return lib.kf_paged_attention(*[null] * 7, starts, *[null] * 3, 0, tokens, B, blocks, width, Hq, Hkv, D, T,
                                      *qs, mq, mc, scale, 1, 3, dtype, cdt, null)

    for bad in (dict(B=0), dict(Hkv=0), dict(Hq=3), dict(D=72), dict(D=272), dict(D=0), dict(T=8), dict(T=48),
                dict(blocks=0), dict(width=0), dict(mq=0), dict(mc=-1), dict(tokens=-1), dict(tokens=5),
                dict(scale=0.0), dict(scale=math.inf), dict(dtype=_lib.KF_F32), dict(dtype=7), dict(cdt=2), dict()):
        assert attn(**bad) == 1, bad
        assert b"kf_paged_attention" in lib.kf_last_error()
    assert attn(tokens=1 << 31, starts=ctypes.c_void_p(16)) == 2
    assert attn(tokens=0, starts=ctypes.c_void_p(16)) == 0
    assert lib.kf_paged_attention_workspace_bytes(4, 4, 4, 3, 64, 1, 64) == -1

    def app(tokens=4, blocks=8, Hkv=2, D=64, T=16, strides=(128, 64, 128, 64), dtype=_lib.KF_F16, cdt=0):
        return lib.kf_paged_cache_append(*[null] * 7, tokens, blocks, Hkv, D, T, *strides, dtype, cdt, null)

    for bad in (dict(tokens=-1), dict(blocks=0), dict(Hkv=0), dict(D=8), dict(T=256), dict(dtype=0), dict(cdt=-1), dict()):
        assert app(**bad) == 1, bad
        assert b"kf_paged_cache_append" in lib.kf_last_error()
    assert app(blocks=1 << 31) == 2
    assert app(tokens=0) == 0

    def tab(B=2, width=4, free=4, total=4, T=16):
        return lib.kf_paged_block_tables(*[null] * 9, B, width, free, total, T, null)

    for bad in (dict(B=0), dict(width=-1), dict(free=-1), dict(total=-1), dict(T=0), dict()):
        assert tab(**bad) == 1, bad
        assert b"kf_paged_block_tables" in lib.kf_last_error()
    assert tab(B=4097) == 2
    assert tab(total=(1 << 30) + 1) == 2


def test_c_entries_refuse_what_no_launch_holds():
    """A launch has less than 2^32 threads."""
    lib = _lib.load()
    null, some = ctypes.c_void_p(0), ctypes.c_void_p(16)
    assert lib.kf_paged_cache_append(*[null] * 7, 1 << 27, 8, 2, 64, 16, 128, 64, 128, 64, _lib.KF_F16, 0, null) == 2
    assert b"2^27" in lib.kf_last_error()
    many = (1 << 22, 1 << 20, 8, 8, 64, 200, 64)  # tokens, requests, heads, key heads, dim, longest, context
    assert lib.kf_paged_attention_workspace_bytes(*many) == -1
    assert b"too many requests of many rows" in lib.kf_last_error()
    assert lib.kf_paged_attention(*[null] * 7, some, *[null] * 3, 0, *many[:2], 8, 4, 8, 8, 64, 16, 512, 64, 200, 64, 0.1, 1,
                                  3, _lib.KF_BF16, 1, null) == 2
    assert lib.kf_paged_attention_workspace_bytes(4, 4, 4, 2, 64, 1 << 62, 64) == -1  # and no product wraps


@pytest.mark.parametrize("max_query_len", [1, 128, 129, 4096])
@pytest.mark.parametrize("Hq,Hkv,D", [(1, 1, 16), (32, 8, 128), (64, 1, 256)])
def test_workspace_of_any_sound_shape(Hq, Hkv, D, max_query_len):
    """Never negative, and at most four parts of 128 rows for each of 256 CUs,
    whatever the lengths; no tokens included."""
    lib = _lib.load()
    for tokens in (0, 1, 127, 128, 129, 5000):
        for B in (1, 3, 700):
            for context in (0, 1, 128, 1024, 2049, 2 ** 31 - 1):
                got = lib.kf_paged_attention_workspace_bytes(tokens, B, Hq, Hkv, D, max_query_len, context)
                assert 0 <= got <= 4 * 256 * 128 * (D * 4 + 8)


def test_bad_pages_lead_nowhere():
    """The index arithmetic of the kernels, on the host: no table entry, slot,
    start or length leads outside the arrays."""
    lib = _lib.load()
    worst = [-2 ** 31, -1, 0, 5, 7, 8, 2 ** 31 - 1]
    table = (ctypes.c_int32 * len(worst))(*worst)
    for shift in (4, 5, 7):
        per = 1 << (shift - 4)
        for group in [*range(len(worst) * per + 3), 2 ** 27, (2 ** 31 - 1) // 16]:
            got = lib.kfm_paged_block_of_group(table, len(worst), 8, shift, group)
            entry = worst[group // per] if group // per < len(worst) else -1
            assert got == (entry if 0 <= entry < 8 else -1)
    for slot in (-2 ** 63, -1, 0, 127, 128, 2 ** 62):
        assert lib.kfm_paged_block_of_slot(slot, 128, 4) == (slot // 16 if 0 <= slot < 128 else -1)

    result = (ctypes.c_int32 * 4)()
    for starts in ((0, 5), (5, 0), (-7, 3), (2, 2 ** 31 - 1), (2 ** 31 - 1, 2 ** 31 - 1), (-2 ** 31, -2 ** 31)):
        for context in (-2 ** 31, -1, 0, 1, 100, 2 ** 31 - 1):
            for causal in (0, 1):
                lib.kfm_paged_request((ctypes.c_int32 * 2)(*starts), (ctypes.c_int32 * 1)(context), 0, 10, 0, causal,
                                      result)
                first, n, ctx, seen = result
                assert 0 <= first <= first + n <= 10
                assert 0 <= ctx <= 2 ** 31 - 256 and 0 <= seen <= ctx + 1
                assert seen == max(0, ctx - n + 1 if causal else ctx)
    lib.kfm_paged_request(None, (ctypes.c_int32 * 3)(4, 5, 6), 2, 3, 0, 1, result)
    assert list(result) == [2, 1, 6, 6]


# ---------------------------------------------------------------------------
# The oracle against independent statements.
# ---------------------------------------------------------------------------
def test_oracle_codes_are_the_nearest():
    every = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    every = every[torch.isfinite(every)].unique()
    y = torch.cat([torch.linspace(-500, 500, 4001, dtype=torch.float64), torch.logspace(-5, 3, 801, dtype=torch.float64),
                   (every[1:] + every[:-1]) / 2])
    got = orc.round_code(y, torch.float8_e4m3fn)
    assert torch.isin(got, every).all()
    nearest = (y.clamp(-448, 448)[:, None] - every).abs().min(1).values
    assert torch.equal((got - y.clamp(-448, 448)).abs(), nearest)
    assert torch.equal(got, y.clamp(-448, 448).float().to(torch.float8_e4m3fn).double())  # ties to even, as torch


@pytest.mark.parametrize("most", [448.0, 127.0])
def test_oracle_scale_is_the_least_that_fits(most):
    for a in (0.0, 1e-45, 1e-38, 0.3, most, most * (1 + 2.0 ** -20), most / 2, 65504.0, 3.3e38):
        s = orc.scale_of(a, most)
        assert a <= most * s and math.log2(s) == int(math.log2(s))
        assert s == 2.0 ** -126 or a > most * s / 2


@pytest.mark.parametrize("causal", [False, True])
def test_oracle_attention_is_the_dense_attention(causal):
    """Whole blocks in order and unit scales: the paged result is fa.attention's."""
    g = torch.Generator().manual_seed(3)
    T, H, D, c, n = 16, 2, 32, 32, 5
    key = torch.randint(-127, 128, (2, H, T, D), generator=g).to(torch.int8)
    value = torch.randint(-127, 128, (2, H, T // 16, D, 16), generator=g).to(torch.int8)
    scales = torch.full((2, H), 0.01)
    q = torch.randn(n, 4, D, generator=g)
    out, lse, *_ = orc.attention(q, (key, value, scales, scales), [[0, 1]], [c], [0, n], causal=causal)
    k = key.double().transpose(1, 2).reshape(1, c, H, D) * scales.double()[0, 0]
    v = orc.tokens_of(value.double()).transpose(1, 2).reshape(1, c, H, D) * scales.double()[0, 0]
    want = ofa.attention(q[None].double(), k, v, causal=causal)
    torch.testing.assert_close(out[None], want, rtol=1e-12, atol=1e-12)
    torch.testing.assert_close(lse[None], ofa.attention_lse(q[None].double(), k, causal=causal), rtol=1e-12, atol=1e-12)


def test_oracle_tables():
    tables, starts, context, slots, used = orc.block_tables(
        [[9, -1, -1], [-1] * 3, [5, 6, -1]], [3, 0, 32], [14, 0, 1], [20, 21, 22], 1, 17, 16)
    assert tables == [[9, 21, -1], [-1, -1, -1], [5, 6, 22]]
    assert (starts, context, used) == ([0, 14, 14, 15], [17, 0, 33], 3)
    assert slots == [9 * 16 + p for p in range(3, 16)] + [21 * 16] + [22 * 16] + [-1, -1]
