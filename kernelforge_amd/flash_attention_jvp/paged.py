"""Attention over a paged key/value cache held in 8 bits, and what keeps it.

The serving side of ``flash_attention``: the keys and values of earlier tokens
stay on the GPU in blocks of 16 to 128 tokens, in e4m3 or int8 with one fp32
scale for each block and head, and requests of any length share the blocks
through tables.  Three operators, all of them on the current stream, without a
host synchronisation and safe to capture:

- ``paged_block_tables_``   a step's block tables, query starts and slots, from
  the lengths (``kf_paged_block_tables``)
- ``paged_cache_append_``   the new keys and values into their slots
  (``kf_paged_cache_append``)
- ``paged_attention``       the new queries over the cached keys
  (``kf_paged_attention``)

A step of a serving loop:

    cache = paged_kv_cache(num_blocks, num_kv_heads, head_dim)
    ...
    starts, context, slots, used = paged_block_tables_(
        tables, context, new_tokens, free_blocks, used, total_tokens=n, block_tokens=16)
    paged_cache_append_(cache, k, v, slots)                  # k, v [n, Hkv, D]
    out = paged_attention(q, cache, tables, context, starts) # q [n, Hq, D]

The reference has no cache; rows without a key follow its forward's convention
(out 0, LSE +inf; flash_attention_jvp/custom.py:70-71).
"""

from __future__ import annotations

import contextlib
import math
from functools import lru_cache
from typing import NamedTuple

import torch

from .. import _lib

_CACHE_DTYPES = {torch.float8_e4m3fn: _lib.KF_CACHE_E4M3, torch.int8: _lib.KF_CACHE_INT8}
_BLOCK_TOKENS = (16, 32, 64, 128)
_NULL = contextlib.nullcontext()


class PagedKVCache(NamedTuple):
    """The cache's four tensors (any 4-tuple of such tensors serves).

    key ``[blocks, Hkv, T, D]`` and value ``[blocks, Hkv, T/16, D, 16]`` (the 16
    tokens of a group innermost) in e4m3 or int8, T the block's tokens; fp32
    scales ``[blocks, Hkv]``, none negative.  An element is its code times its scale.
    """

    key: torch.Tensor
    value: torch.Tensor
    key_scale: torch.Tensor
    value_scale: torch.Tensor


def paged_kv_cache(num_blocks: int, num_kv_heads: int, head_dim: int, *, block_tokens: int = 16,
                   dtype: torch.dtype = torch.float8_e4m3fn, device="cuda") -> PagedKVCache:
    """An empty cache: every code and scale 0."""
    if min(num_blocks, num_kv_heads) < 1:
        raise ValueError("num_blocks and num_kv_heads must be positive")
    _check_layout(head_dim, block_tokens, dtype)

    def zeros(*shape):
        return torch.zeros(shape, dtype=torch.uint8, device=device).view(dtype)

    scales = [torch.zeros(num_blocks, num_kv_heads, dtype=torch.float32, device=device) for _ in range(2)]
    return PagedKVCache(zeros(num_blocks, num_kv_heads, block_tokens, head_dim),
                        zeros(num_blocks, num_kv_heads, block_tokens // 16, head_dim, 16), *scales)


def _check_layout(head_dim, block_tokens, dtype):
    if head_dim % 16 or not 16 <= head_dim <= 256:
        raise ValueError("the head dim must be a multiple of 16 <= 256")
    if block_tokens not in _BLOCK_TOKENS:
        raise ValueError(f"block_tokens must be one of {_BLOCK_TOKENS}")
    if dtype not in _CACHE_DTYPES:
        raise ValueError("the cache's dtype must be float8_e4m3fn or int8")


def _check_cache(cache, device):
    """(blocks, Hkv, T, D) of a cache whose tensors all fit one another."""
    key, value, key_scale, value_scale = cache
    shape = key.shape
    if len(shape) != 4 or 0 in shape:
        raise ValueError("the key cache must have shape [blocks, heads, block_tokens, dim]")
    blocks, heads, T, D = shape
    dtype = key.dtype
    _check_layout(D, T, dtype)
    if value.shape != (blocks, heads, T // 16, D, 16) or value.dtype != dtype:
        raise ValueError("the value cache must have shape [blocks, heads, block_tokens / 16, dim, 16] and the keys' dtype")
    pair = (blocks, heads)
    f32 = torch.float32
    if (key_scale.shape != pair or key_scale.dtype != f32 or value_scale.shape != pair or value_scale.dtype != f32):
        raise ValueError("the cache's scales must be float32 [blocks, heads]")
    if not (key.is_contiguous() and value.is_contiguous() and key_scale.is_contiguous()
            and value_scale.is_contiguous()):
        raise ValueError("the cache's tensors must be contiguous")
    if (key.device != device or value.device != device or key_scale.device != device
            or value_scale.device != device):
        raise ValueError("the cache must be on the call's device")
    return blocks, heads, T, D


def _check_ints(name, t, shape, dtype, device):
    if t.dtype != dtype or t.shape != shape:
        raise ValueError(f"{name} must be {str(dtype).removeprefix('torch.')} of shape {tuple(shape)}, "
                         f"got {t.dtype} {tuple(t.shape)}")
    if t.device != device or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous and on the call's device")


def _check_no_grad(*tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t.requires_grad:
                raise RuntimeError("the paged operators have no backward: call them under torch.no_grad()")


def _rows(t: torch.Tensor):
    """t [tokens, heads, D] and its strides of tokens and heads, where its rows can
    be read as 16-byte vectors (a part of a packed projection can), else a copy's."""
    st, sh, sd = t.stride()
    if sd == 1 and st % 8 == 0 and st < 1 << 26 and sh % 8 == 0 and t.data_ptr() % 16 == 0:
        return t, st, sh
    # (a contiguous tensor's clone keeps the strides of its dimensions of one)
    t = torch.empty(t.shape, dtype=t.dtype, device=t.device).copy_(t)
    return t, *t.stride()[:2]


def _on(index: int):
    """Makes a device current for a launch (nothing to do where it is)."""
    return _NULL if torch._C._cuda_getDevice() == index else torch.cuda.device(index)


def paged_block_tables_(block_tables, context_lens, query_lens, free_blocks, free_used, *, total_tokens: int,
                        block_tokens: int, in_place: bool = False):
    """Extend every request's table for its new tokens; returns
    ``(query_starts, context_lens, slots, free_used)``.

    block_tables int32 ``[B, W]`` is updated in place: a request with
    ``context_lens[b]`` cached and ``query_lens[b]`` new tokens gets the blocks it
    lacks from ``free_blocks[free_used:]`` (int32 ids, in order of b); its other
    entries keep their values.  Returned: query_starts int32 ``[B + 1]``, the
    lengths with the new tokens int32 ``[B]``, slots int64 ``[total_tokens]`` for
    ``paged_cache_append_``, and the advanced count int32 ``[1]`` of taken blocks.
    With ``in_place`` the lengths and the count are written into ``context_lens``
    and ``free_used`` themselves (for a captured step that is replayed).

    total_tokens is the step's token buffer: slots behind the last request's
    tokens are -1, and tokens past the buffer are not taken.  A token whose table
    is too narrow or for whom no block is left gets slot -1 (and a table entry of
    -1, at which ``paged_attention`` gives NaN); ``free_used`` then exceeds
    ``len(free_blocks)``, where a caller sees it.  At most 4096 requests.
    """
    if block_tables.ndim != 2 or block_tables.dtype != torch.int32:
        raise ValueError("block_tables must be int32 [requests, width]")
    if block_tokens not in _BLOCK_TOKENS:
        raise ValueError(f"block_tokens must be one of {_BLOCK_TOKENS}")
    if total_tokens < 0:
        raise ValueError("total_tokens must be >= 0")
    B, width = block_tables.shape
    if B < 1:
        raise ValueError("block_tables must hold a request")
    if free_blocks.ndim != 1:
        raise ValueError("free_blocks must be int32 of one dimension")
    device = block_tables.device
    i32 = torch.int32
    _check_ints("block_tables", block_tables, (B, width), i32, device)
    _check_ints("context_lens", context_lens, (B,), i32, device)
    _check_ints("query_lens", query_lens, (B,), i32, device)
    _check_ints("free_blocks", free_blocks, free_blocks.shape, i32, device)
    _check_ints("free_used", free_used, (1,), i32, device)
    _lib.require_gpu(block_tables)
    slots = torch.empty(total_tokens, dtype=torch.int64, device=device)
    if in_place:
        starts, context, used = torch.empty(B + 1, dtype=i32, device=device), context_lens, free_used
    else:  # parts of one allocation (an allocation takes the host 1.2 us, as the split does)
        starts, context, used = torch.empty(2 * B + 2, dtype=i32, device=device).split_with_sizes((B + 1, B, 1))
    with _on(device.index):
        rc = _lib.load().kf_paged_block_tables(
            block_tables.data_ptr(), context_lens.data_ptr(), query_lens.data_ptr(), free_blocks.data_ptr(),
            free_used.data_ptr(), starts.data_ptr(), context.data_ptr(), slots.data_ptr(), used.data_ptr(), B, width,
            free_blocks.shape[0], total_tokens, block_tokens, _lib.stream_of(block_tables))
    _lib.check(rc, "kf_paged_block_tables")
    return starts, context, slots, used


def paged_cache_append_(cache, key, value, slots):
    """Write new keys and values ``[tokens, Hkv, D]`` (fp16 or bf16) into their
    slots (int64 ``[tokens]``, from ``paged_block_tables_``); returns the cache.

    A block's scale for a head is the least power of two with which its largest
    element fits (448 in e4m3, 127 in int8) and grows as larger elements arrive:
    the codes that the block holds are then scaled down with it.  Powers of two
    keep every quotient exact, so an element is rounded once, and an e4m3 code
    loses nothing when its block's scale grows (above its subnormals).  Writing a
    block's first slot starts the block: what it held is dropped.  An infinity or
    NaN makes the scale NaN, and every row that reads the block, until then.

    Slots outside the cache are skipped.  The tokens of one block must follow one
    another, as the tokens of one request do; of two that name one slot the later
    is kept.  key and value may be parts of a packed projection
    (``qkv[:, Hq:Hq + Hkv]``).
    """
    if key.ndim != 3 or key.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError("key must be float16 or bfloat16 of shape [tokens, heads, dim]")
    if value.shape != key.shape or value.dtype != key.dtype or value.device != key.device:
        raise ValueError("value must have key's shape, dtype, and device")
    device = key.device
    blocks, heads, T, D = _check_cache(cache, device)
    tokens = key.shape[0]
    if key.shape[1:] != (heads, D):
        raise ValueError(f"key must have the cache's {heads} heads of {D}")
    _check_ints("slots", slots, (tokens,), torch.int64, device)
    _lib.require_gpu(key)
    _check_no_grad(key, value)
    if tokens == 0:
        return cache
    (key, key_ts, key_hs), (value, value_ts, value_hs) = _rows(key), _rows(value)
    kc, vc, ks, vs = cache
    with _on(device.index):
        rc = _lib.load().kf_paged_cache_append(
            key.data_ptr(), value.data_ptr(), slots.data_ptr(), kc.data_ptr(), vc.data_ptr(), ks.data_ptr(),
            vs.data_ptr(), tokens, blocks, heads, D, T, key_ts, key_hs, value_ts, value_hs, _lib.kf_dtype(key.dtype),
            _CACHE_DTYPES[kc.dtype], _lib.stream_of(key))
    _lib.check(rc, "kf_paged_cache_append")
    return cache


@lru_cache(maxsize=4096)
def _workspace_bytes(device_index: int, *shape) -> int:
    """``kf_paged_attention_workspace_bytes`` of a shape on a device (the current one)."""
    return int(_lib.load().kf_paged_attention_workspace_bytes(*shape))


def paged_attention(q, cache, block_tables, context_lens, query_starts=None, *, max_query_len: int | None = None,
                    max_context_len: int | None = None, softmax_scale: float | None = None, causal: bool = True,
                    return_lse: bool = False, out: torch.Tensor | None = None):
    """Attention of new tokens over the cached keys of their requests.

    q ``[tokens, Hq, D]`` (fp16 or bf16) holds the requests' new tokens one
    request after the other: those of request b are ``query_starts[b]`` to
    ``query_starts[b + 1] - 1`` (int32 ``[B + 1]``); without ``query_starts`` every
    request has one.  block_tables int32 ``[B, W]``; context_lens int32 ``[B]``
    counts the cached tokens, the new ones included (append them first).  Query
    head h reads key head ``h // (Hq / Hkv)``.  causal: the new tokens stand at
    the context's end and see no later key.

    Returns out ``[tokens, Hq, D]`` and, with ``return_lse``, the fp32 natural-log
    LSE ``[Hq, tokens]``.  A row that sees no key gives 0 and +inf; one that sees a
    table entry outside the cache, or a key past the table, gives NaN.  Rows of
    tokens behind the last request are 0 (+inf), or left as they were in a
    caller's ``out``.

    max_query_len bounds the new tokens of a request (default: all of q's) and
    has to hold: the queries of a request past it give NaN.  max_context_len
    (default: the table's width) only guides how the keys are split over
    workgroups.  out may be q itself, and overlap nothing else.  Results do not depend on the rest of the batch beyond the last
    place, and are the same at every repeat.  There is no backward.
    """
    if q.ndim != 3 or q.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError("q must be float16 or bfloat16 of shape [tokens, heads, dim]")
    device = q.device
    blocks, Hkv, T, D = _check_cache(cache, device)
    tokens, Hq, dim = q.shape
    if dim != D or Hq < 1 or Hq % Hkv:
        raise ValueError("q must have the cache's head dim and a multiple of its heads")
    table_shape = block_tables.shape
    if len(table_shape) != 2 or 0 in table_shape:
        raise ValueError("block_tables must be int32 [requests, width], neither of them 0")
    B, width = table_shape
    i32 = torch.int32
    _check_ints("block_tables", block_tables, table_shape, i32, device)
    _check_ints("context_lens", context_lens, (B,), i32, device)
    if query_starts is not None:
        _check_ints("query_starts", query_starts, (B + 1,), i32, device)
    elif tokens != B:
        raise ValueError("without query_starts q must hold one token of every request")
    scale = D ** -0.5 if softmax_scale is None else float(softmax_scale)
    if not math.isfinite(scale) or scale <= 0:
        raise ValueError("softmax_scale must be finite and positive")
    if query_starts is None:
        max_query_len = 1
    elif max_query_len is None:
        max_query_len = tokens
    elif max_query_len < 1:
        raise ValueError("max_query_len must be positive")
    if max_context_len is None:
        max_context_len = width * T
    elif max_context_len < 0:
        raise ValueError("max_context_len must be >= 0")
    if out is not None and (out.shape != q.shape or out.dtype != q.dtype or out.device != device
                            or not out.is_contiguous() or out.data_ptr() % 16):
        raise ValueError("out must be contiguous and have q's shape, dtype, and device")
    _lib.require_gpu(q)
    given = out is not None
    if given:
        _check_no_grad(q, out)
    else:
        _check_no_grad(q)
        out = torch.empty(tokens, Hq, D, dtype=q.dtype, device=device)
    lse = torch.empty((Hq, tokens), dtype=torch.float32, device=device) if return_lse else None
    if tokens == 0:
        return (out, lse) if return_lse else out
    q, q_ts, q_hs = _rows(q)
    kc, vc, ks, vs = cache
    if max_query_len > tokens:
        max_query_len = tokens
    if max_context_len > width * T:
        max_context_len = width * T
    index = device.index
    with _on(index):
        nbytes = _workspace_bytes(index, tokens, B, Hq, Hkv, D, max_query_len, max_context_len)
        if nbytes < 0:
            raise ValueError(f"paged_attention: {_lib.load().kf_last_error().decode()}")
        ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
        rc = _lib.load().kf_paged_attention(
            q.data_ptr(), kc.data_ptr(), vc.data_ptr(), ks.data_ptr(), vs.data_ptr(), block_tables.data_ptr(),
            context_lens.data_ptr(), None if query_starts is None else query_starts.data_ptr(), out.data_ptr(),
            None if lse is None else lse.data_ptr(), None if ws is None else ws.data_ptr(), nbytes, tokens, B, blocks,
            width, Hq, Hkv, D, T, q_ts, q_hs, max_query_len, max_context_len, scale, bool(causal), 2 if given else 3,
            _lib.kf_dtype(q.dtype), _CACHE_DTYPES[kc.dtype], _lib.stream_of(q))
    _lib.check(rc, "kf_paged_attention")
    return (out, lse) if return_lse else out
