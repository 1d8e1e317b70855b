"""The paged 8-bit key/value cache and the attention over it, as a serving loop runs them.

``listed()`` names the cases, ``draw(rng)`` gives one more of the same ranges;
``prepare`` makes a case's inputs on the GPU from a seed, ``run`` is one pass:
where ``own`` is false in elementary torch operations, where it is true through
the framework's entry points.  ``work`` is the bytes and operations a pass
cannot do without, ``exact`` the result in 64 bits.

A case's ``path`` is one of
  tables     ``paged_block_tables_``: from each request's cached and new token
             counts the block tables, the query starts and every token's slot
  append     ``paged_cache_append_``: new keys and values into their slots, in 8
             bits with a power-of-two scale for each block of tokens and head
  attention  ``paged_attention``: the new tokens' queries over the cached keys

A cache is ``(key[blocks, Hkv, block, D], value[blocks, Hkv, block / 16, D, 16],
key_scale[blocks, Hkv], value_scale[blocks, Hkv])``: a value group holds 16
tokens, the token innermost.  ``context`` counts a request's cached tokens,
``queries`` its new ones, which stand at the end of the context.

The caches come back as they are held, codes and scales.  A scale is a power of
two, so every quotient is exact and a code is that quotient rounded once: any
correct implementation holds the same codes.
"""

import math
import random

import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16}
CACHES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
LARGEST = {"e4m3": 448.0, "int8": 127.0}


def _tables(name, B, block, queries, context, width, spare=0):
    return dict(name=name, path="tables", B=B, block=block, qmin=queries[0], qmax=queries[1], cmin=context[0],
                cmax=context[1], width=width, spare=spare, lens=1)


def _append(name, B, Hkv, D, block, queries, context, cache, dtype="bfloat16", packed=False):
    return dict(name=name, path="append", B=B, Hkv=Hkv, D=D, block=block, qmin=queries[0], qmax=queries[1],
                cmin=context[0], cmax=context[1], cache=cache, dtype=dtype, packed=packed, lens=2)


def _attn(name, B, Hq, Hkv, D, block, queries, context, cache, dtype="bfloat16", causal=True):
    return dict(name=name, path="attention", B=B, Hq=Hq, Hkv=Hkv, D=D, block=block, qmin=queries[0],
                qmax=queries[1], cmin=context[0], cmax=context[1], cache=cache, dtype=dtype, causal=causal, lens=3)


def listed():
    return [
        # One decoding step's bookkeeping for a batch of requests: latency.
        _tables("tables_decode", 64, 16, (1, 1), (1, 8192), 513),
        # A batch of prompts admitted at once, ragged, some behind a cached
        # prefix; the token buffer is longer than the prompts.
        _tables("tables_prompts", 48, 16, (100, 4096), (100, 4096), 320, spare=1000),
        # One new token for each request of a decoding batch.
        _append("append_decode", 64, 8, 128, 16, (1, 1), (1, 1024), "e4m3"),
        # The prompts of a large batch: memory bandwidth.
        _append("append_prompts", 5, 8, 128, 16, (2500, 4096), (2500, 4096), "e4m3", packed=True),
        # Chunks that begin inside a block, narrow heads, int8 and wide blocks.
        _append("append_chunks", 7, 16, 64, 64, (33, 700), (100, 3001), "int8", "float16"),
        # One request's next token against a short context: latency.
        _attn("decode_short", 1, 16, 16, 64, 16, (1, 1), (333, 333), "int8"),
        # A decoding batch with grouped heads and ragged contexts: bandwidth.
        _attn("decode_batch", 32, 32, 8, 128, 16, (1, 1), (500, 8192), "e4m3"),
        # Two requests over very long contexts: the work is along one axis.
        _attn("decode_long", 2, 32, 8, 128, 64, (1, 1), (60000, 100001), "e4m3", "float16"),
        # Every query head on one key head of the widest dim.
        _attn("decode_wide", 16, 16, 1, 256, 32, (1, 1), (1000, 16384), "int8"),
        # A few new tokens of each request (drafts that are checked at once).
        _attn("verify_drafts", 8, 32, 8, 128, 16, (4, 4), (1000, 8192), "int8"),
        # The next chunk of two long prompts: matrix products.
        _attn("prompt_chunk", 2, 32, 8, 128, 16, (2048, 2048), (6000, 8192), "e4m3"),
        # Decoding and ragged prompts in one call, at a head dim of 80.
        _attn("mixed_batch", 12, 16, 4, 80, 16, (1, 700), (64, 3001), "e4m3", "float16"),
    ]


def _logint(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 8e12, w["flops"] / 2.5e15)


def draw(rng):
    """One more case of the ranges the listed ones stand for."""
    most = max(_cost(c) for c in listed())
    while True:
        case = _draw(rng)
        case.pop("name", None)
        case["lens"] = rng.randrange(1 << 20)
        # The plain form's scores of the padded batch have to fit beside three states.
        scores = case.get("Hq", 0) * case["B"] * case["qmax"] * case["cmax"]
        if _cost(case) <= most and scores <= 2e9:
            return case


def _draw(rng):
    path = rng.choice(["tables", "append", "append", "decode", "decode", "decode", "few", "chunk"])
    block = rng.choice([16, 16, 16, 32, 64, 128])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16"])
    cache = rng.choice(["e4m3", "e4m3", "int8"])
    if path == "tables":
        B = _logint(rng, 1, 512)
        hi = _logint(rng, 1, 65536 // B)
        lo = max(1, int(hi * rng.random()))
        ctx = (lo, hi + _logint(rng, 1, 8192))
        return _tables("", B, block, (lo, hi), ctx, -(-ctx[1] // block) + rng.randrange(8), spare=rng.choice([0, 0, 7, 500]))
    D = rng.choice([64, 64, 128, 128, 128, 80, 96, 256, 16, 112])
    Hkv = rng.choice([1, 2, 4, 8, 16])
    if path == "append":
        B = _logint(rng, 1, 128)
        hi = _logint(rng, 1, 16384 // B)
        lo = max(1, int(hi * rng.random()))
        return _append("", B, Hkv, D, block, (lo, hi), (lo, hi + _logint(rng, 1, 1000)), cache, dtype,
                       rng.random() < 0.5)
    Hq = Hkv * rng.choice([1, 2, 4, 8, 3])
    if path == "decode":
        B = _logint(rng, 1, 64)
        hi = _logint(rng, 16, 120000 // B)
        return _attn("", B, Hq, Hkv, D, block, (1, 1), (max(1, int(hi * rng.random())), hi), cache, dtype)
    B = _logint(rng, 1, 16)
    if path == "few":
        hi = _logint(rng, 200, 60000 // B)
        n = _logint(rng, 2, 40)
        return _attn("", B, Hq, Hkv, D, block, (rng.choice([1, n]), n), (max(n, int(hi * rng.random())), hi + n), cache,
                     dtype, rng.random() < 0.8)
    n = _logint(rng, 41, 6000 // B)
    hi = n + _logint(rng, 1, 8000 // B)
    return _attn("", B, Hq, Hkv, D, block, (rng.choice([1, n]), n), (n, hi), cache, dtype, rng.random() < 0.8)


# ---------------------------------------------------------------------------
# Lengths and inputs.
# ---------------------------------------------------------------------------
def _lengths(case):
    """Each request's (new tokens, tokens in all after them)."""
    rng = random.Random(case["lens"])
    got = []
    for b in range(case["B"]):
        q = _logint(rng, case["qmin"], case["qmax"]) if b else case["qmax"]
        c = rng.randint(max(q, case["cmin"]), max(q, case["cmax"])) if b else case["cmax"]
        got.append((q, c))
    return got


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _starts(lengths):
    starts = [0]
    for q, _ in lengths:
        starts.append(starts[-1] + q)
    return starts


def _new_blocks(case):
    """Blocks that the new tokens of each request take from the free list."""
    T = case["block"]
    return [-(-c // T) - -(-(c - q) // T) for q, c in _lengths(case)]


def _paged(lengths, block, g, width=None):
    """Random block ids for every request's context: (tables, number of blocks)."""
    need = [-(-c // block) for _, c in lengths]
    width = width or max(need)
    blocks = sum(need)
    ids = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)
    owner = torch.repeat_interleave(torch.arange(len(need), device="cuda"), _ints(need, torch.int64))
    first = _ints([sum(need[:b]) for b in range(len(need))], torch.int64)
    tables = torch.full((len(need), width), -1, dtype=torch.int32, device="cuda")
    tables[owner, torch.arange(blocks, device="cuda") - first[owner]] = ids
    return tables, blocks


def _codes(x, cache):
    """Elements in the cache's type, rounded to the nearest."""
    x = x.clamp(-LARGEST[cache], LARGEST[cache])
    return (x.round() if cache == "int8" else x).to(CACHES[cache])


def _random_cache(blocks, case, g):
    """A filled cache: keys with a few strong channels, values whose size varies
    from block to block."""
    Hkv, D, T, cache = case["Hkv"], case["D"], case["block"], case["cache"]
    strong = torch.ones(Hkv, 1, D, device="cuda")
    strong[:, :, 3::29] = 4.0
    got = []
    for part in range(2):
        codes = torch.empty(blocks, Hkv, T, D, dtype=CACHES[cache], device="cuda")
        scales = torch.empty(blocks, Hkv, device="cuda")
        for i in range(0, blocks, 4096):
            n = min(4096, blocks - i)
            x = torch.randn(n, Hkv, T, D, generator=g, device="cuda")
            x *= strong if part == 0 else torch.exp(0.7 * torch.randn(n, Hkv, 1, 1, generator=g, device="cuda"))
            s = _power_of_two(x.abs().amax((2, 3)), cache)
            codes[i:i + n] = _codes(x / s[:, :, None, None], cache)
            scales[i:i + n] = s
        got += [codes, scales]
    key, key_scale, value, value_scale = got
    value = value.view(torch.uint8).reshape(blocks, Hkv, T // 16, 16, D).transpose(-1, -2).contiguous()
    return key, value.view(CACHES[cache]), key_scale, value_scale


def _empty_cache(blocks, case):
    Hkv, D, T, dt = case["Hkv"], case["D"], case["block"], CACHES[case["cache"]]
    zeros = [torch.zeros(shape, dtype=torch.uint8, device="cuda").view(dt)
             for shape in ((blocks, Hkv, T, D), (blocks, Hkv, T // 16, D, 16))]
    return (*zeros, torch.zeros(blocks, Hkv, device="cuda"), torch.zeros(blocks, Hkv, device="cuda"))


def _new_tokens(case, seed):
    """Keys and values of the new tokens; packed: parts of one qkv tensor, as a
    projection leaves them."""
    g = torch.Generator("cuda").manual_seed(seed + 1)
    T = _starts(_lengths(case))[-1]
    Hkv, D, dt = case["Hkv"], case["D"], DTYPES[case["dtype"]]
    heads = 4 * Hkv if case["packed"] else 2 * Hkv
    kv = torch.randn(T, heads, D, generator=g, device="cuda")
    kv *= torch.exp(0.7 * torch.randn(T, heads, 1, generator=g, device="cuda"))
    kv = kv.to(dt)
    return kv[:, heads - 2 * Hkv:heads - Hkv], kv[:, heads - Hkv:]


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    lengths = _lengths(case)
    path, T = case["path"], case["block"]
    state = dict(case=case)
    if path == "tables":
        tables, held = _paged([(0, c - q) for q, c in lengths], T, g, case["width"])
        need = sum(_new_blocks(case))
        used = int(seed) % 5
        free = held + torch.randperm(need + used + 100, generator=g, device="cuda").to(torch.int32)
        return state | dict(tables=tables, context=_ints([c - q for q, c in lengths]),
                            queries=_ints([q for q, _ in lengths]), free=free, used=_ints([used]),
                            total=_starts(lengths)[-1] + case["spare"])
    tables, blocks = _paged(lengths, T, g)
    starts = _starts(lengths)
    if path == "append":
        pos = torch.cat([torch.arange(c - q, c, device="cuda") for q, c in lengths])
        owner = torch.repeat_interleave(torch.arange(len(lengths), device="cuda"),
                                        _ints([q for q, _ in lengths], torch.int64))
        slots = tables[owner, pos // T].long() * T + pos % T
        key, value = _new_tokens(case, seed)
        cache = _random_cache(blocks, case, g)
        return state | dict(cache=cache, key=key, value=value, slots=slots)
    q = torch.randn(starts[-1], case["Hq"], case["D"], generator=g, device="cuda").to(DTYPES[case["dtype"]])
    return state | dict(q=q, cache=_random_cache(blocks, case, g), tables=tables, context=_ints([c for _, c in lengths]),
                        starts=None if case["qmax"] == 1 else _ints(starts), longest=max(c for _, c in lengths))


# ---------------------------------------------------------------------------
# One pass.
# ---------------------------------------------------------------------------
def run(state):
    case, path = state["case"], state["case"]["path"]
    if own:
        from kernelforge_amd.flash_attention_jvp import paged_attention, paged_block_tables_, paged_cache_append_

        if path == "tables":
            return state["tables"], *paged_block_tables_(
                state["tables"], state["context"], state["queries"], state["free"], state["used"],
                total_tokens=state["total"], block_tokens=case["block"])
        if path == "append":
            paged_cache_append_(state["cache"], state["key"], state["value"], state["slots"])
            return state["cache"]
        return paged_attention(state["q"], state["cache"], state["tables"], state["context"], state["starts"],
                               max_query_len=case["qmax"], causal=case["causal"], return_lse=True)
    return {"tables": _plain_tables, "append": _plain_append, "attention": _plain_attention}[path](state)


def _plain_tables(s):
    T, total = s["case"]["block"], s["total"]
    tables, free = s["tables"], s["free"]
    old, new = s["context"].long(), s["queries"].long()
    B, width = tables.shape
    starts = torch.cat([new.new_zeros(1), new.cumsum(0)]).clamp(max=total)
    context = old + starts[1:] - starts[:-1]
    held = (old + T - 1) // T
    need = (context + T - 1) // T - held
    first = s["used"] + need.cumsum(0) - need
    j = torch.arange(width, device="cuda")
    fresh = (j >= held[:, None]) & (j < (held + need)[:, None])
    take = (first[:, None] + j - held[:, None]).clamp(0, free.numel() - 1)
    tables = torch.where(fresh, free[take], tables)
    t = torch.arange(total, device="cuda")
    b = torch.searchsorted(starts[1:], t, right=True).clamp(max=B - 1)
    pos = old[b] + t - starts[b]
    ids = tables[b, (pos // T).clamp(max=width - 1)].long()
    slots = torch.where(t < starts[-1], ids * T + pos % T, -1)
    return tables, starts.int(), context.int(), slots, (s["used"] + need.sum()).int()


def _power_of_two(largest, cache):
    """The least power of two s, at least 2^-126, with largest <= LARGEST * s."""
    m, e = torch.frexp(largest.float())
    most, shift = math.frexp(LARGEST[cache])
    e = torch.where(m > most, e + 1, e) - shift
    e = torch.where(largest == 0, -126, e).clamp(-126, 127)
    return ((e + 127) << 23).to(torch.int32).view(torch.float32)


def _plain_append(s):
    T = s["case"]["block"]
    touched, at = torch.unique(s["slots"] // T, return_inverse=True)
    off = s["slots"] % T
    begun = torch.zeros(touched.numel(), dtype=torch.bool, device="cuda").index_fill(0, at[off == 0], True)
    key, value, key_scale, value_scale = s["cache"]
    _plain_write(s["case"], s["key"], key, key_scale, touched, at, off, begun, False)
    _plain_write(s["case"], s["value"], value, value_scale, touched, at, off, begun, True)
    return s["cache"]


def _plain_write(case, x, codes, scales, touched, at, off, begun, grouped):
    """The rows x into rows off of the blocks touched[at], in place; a block that
    is begun forgets what it held.  grouped: 16 tokens innermost."""
    T, Hkv, D, cache = case["block"], case["Hkv"], case["D"], case["cache"]
    n = touched.numel()
    x = x.float()
    largest = torch.zeros(n, Hkv, device="cuda")
    largest.scatter_reduce_(0, at[:, None].expand(-1, Hkv), x.abs().amax(-1), "amax")
    old_scale = torch.where(begun[:, None], 0.0, scales[touched])
    scale = torch.maximum(old_scale, _power_of_two(largest, cache))
    raw = codes.view(torch.uint8)
    held = raw[touched].view(codes.dtype).float()
    if grouped:
        held = held.transpose(-1, -2).reshape(n, Hkv, T, D)
    held = torch.where(begun[:, None, None, None], 0.0, held * (old_scale / scale)[:, :, None, None])
    held[at, :, off] = x / scale[at][:, :, None]
    new = _codes(held, cache).view(torch.uint8)
    if grouped:
        new = new.reshape(n, Hkv, T // 16, 16, D).transpose(-1, -2)
    raw[touched] = new
    scales[touched] = scale


def _gathered(cache, ids, dtype):
    """The keys and values of the blocks ids[B, n], [B, Hkv, n * block, D] each."""
    key, value, key_scale, value_scale = cache
    B, n = ids.shape
    Hkv, T, D = key.shape[1:]
    k = key.view(torch.uint8)[ids].view(key.dtype).to(dtype) * key_scale[ids][..., None, None].to(dtype)
    v = value.view(torch.uint8)[ids].view(key.dtype).to(dtype) * value_scale[ids][..., None, None, None].to(dtype)
    k = k.transpose(1, 2).reshape(B, Hkv, n * T, D)
    v = v.transpose(-1, -2).reshape(B, n, Hkv, T, D).transpose(1, 2).reshape(B, Hkv, n * T, D)
    return k, v


def _plain_attention(s):
    case, q, context = s["case"], s["q"], s["context"].long()
    B, Hq, Hkv, D, T = (case[k] for k in ("B", "Hq", "Hkv", "D", "block"))
    G, Qm = Hq // Hkv, case["qmax"]
    starts = torch.arange(B + 1, device="cuda") if s["starts"] is None else s["starts"].long()
    count = starts[1:] - starts[:-1]
    k, v = _gathered(s["cache"], s["tables"][:, :-(-s["longest"] // T)].clamp(min=0), torch.float32)
    i = torch.arange(Qm, device="cuda")
    live = i < count[:, None]
    at = torch.where(live, starts[:-1, None] + i, 0)
    x = q[at].float().reshape(B, Qm, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * Qm, D)
    scores = (x @ k.transpose(-1, -2).contiguous()).reshape(B, Hkv, G, Qm, -1).mul_(D ** -0.5)
    reach = context[:, None] - (count[:, None] - 1 - i if case["causal"] else 0 * i)
    hidden = torch.arange(k.shape[2], device="cuda") >= reach[..., None]
    scores.masked_fill_(hidden[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = (p.reshape(B, Hkv, G * Qm, -1) @ v).reshape(B, Hkv, G, Qm, D) / total
    lse = (top + total.log()).squeeze(-1).reshape(B, Hq, Qm).transpose(1, 2)[live].T.contiguous()
    return out.permute(0, 3, 1, 2, 4).reshape(B, Qm, Hq, D)[live].to(q.dtype), lse


# ---------------------------------------------------------------------------
# What a pass cannot do without.
# ---------------------------------------------------------------------------
def work(case):
    lengths, T = _lengths(case), case["block"]
    tokens = sum(q for q, _ in lengths)
    if case["path"] == "tables":
        # Lengths in and out, the free blocks taken and written, a slot a token.
        return dict(bytes=16 * case["B"] + 8 * sum(_new_blocks(case)) + 8 * (tokens + case["spare"]), flops=0)
    Hkv, D = case["Hkv"], case["D"]
    if case["path"] == "append":
        # Keys and values in 16 bits in and in 8 out, the slots, both scales of a block.
        blocks = sum(-(-c // T) - (c - q) // T for q, c in lengths)
        return dict(bytes=6 * tokens * Hkv * D + 8 * tokens + 8 * blocks * Hkv, flops=4 * tokens * Hkv * D)
    Hq = case["Hq"]
    pairs = sum(q * (c - q) + q * (q + 1) // 2 if case["causal"] else q * c for q, c in lengths)
    blocks = sum(-(-c // T) for _, c in lengths)
    moved = sum(2 * c * Hkv * D for _, c in lengths) + blocks * (8 * Hkv + 4) + tokens * Hq * (4 * D + 4)
    return dict(bytes=moved, flops=4 * pairs * Hq * D)


# ---------------------------------------------------------------------------
# The results in 64 bits.
# ---------------------------------------------------------------------------
def _rounded(y, cache):
    """float64 rounded to the nearest e4m3 or int8 value, ties to even."""
    y = y.clamp(-LARGEST[cache], LARGEST[cache])
    if cache == "int8":
        return y.round()
    step = torch.exp2(torch.frexp(y)[1].clamp(min=-5).double() - 4)
    return (y / step).round() * step


def _exact_append(case, seed):
    s = prepare(case, seed)
    T, cache = case["block"], case["cache"]
    slots = s["slots"].tolist()
    of = {}
    for t, slot in enumerate(slots):
        of.setdefault(slot // T, []).append(t)
    got = []
    for x, codes, scales, grouped in ((s["key"], s["cache"][0], s["cache"][2], False),
                                      (s["value"], s["cache"][1], s["cache"][3], True)):
        codes, scales = codes.double(), scales.double()
        for block, rows in of.items():
            new = x[rows[0]:rows[-1] + 1].double()
            off = slots[rows[0]] % T
            base = torch.exp2(torch.ceil(torch.log2(new.abs().amax((0, 2)) / LARGEST[cache])).clamp(min=-126))
            held = codes[block].transpose(-1, -2).reshape(-1, T, case["D"]) if grouped else codes[block]
            if off:
                base = torch.maximum(base, scales[block])
                held = held * (scales[block] / base)[:, None, None]
            else:
                held = torch.zeros_like(held)
            held = held.clone()
            held[:, off:off + len(rows)] = (new / base[:, None]).transpose(0, 1)
            held = _rounded(held, cache)
            if grouped:
                held = held.reshape(-1, T // 16, 16, case["D"]).transpose(-1, -2)
            codes[block], scales[block] = held, base
        got.append((codes if cache == "e4m3" else None, scales))
    return got[0][0], got[1][0], got[0][1], got[1][1]


def _exact_attention(case, seed):
    s = prepare(case, seed)
    Hq, Hkv, D, T = (case[k] for k in ("Hq", "Hkv", "D", "block"))
    q = s["q"]
    out = torch.empty(q.shape, dtype=torch.float64, device="cuda")
    lse = torch.empty(Hq, q.shape[0], dtype=torch.float64, device="cuda")
    first = 0
    for b, (n, c) in enumerate(_lengths(case)):
        ids = s["tables"][b, :-(-c // T)].long()
        for h in range(Hkv):
            k = s["cache"][0][ids, h].double() * s["cache"][2][ids, h].double()[:, None, None]
            v = s["cache"][1][ids, h].double() * s["cache"][3][ids, h].double()[:, None, None, None]
            k = k.reshape(-1, D)[:c]
            v = v.transpose(-1, -2).reshape(-1, D)[:c]
            heads = slice(h * Hq // Hkv, (h + 1) * Hq // Hkv)
            x = q[first:first + n, heads].double()
            w = (x.reshape(-1, D) @ k.T.contiguous()).reshape(n, -1, c) / math.sqrt(D)
            if case["causal"]:
                w.masked_fill_((torch.arange(c, device="cuda") > c - n + torch.arange(n, device="cuda")[:, None])[:, None],
                               -math.inf)
            lse[heads, first:first + n] = torch.logsumexp(w, -1).T
            w = torch.softmax(w, -1)
            out[first:first + n, heads] = (w.reshape(-1, c) @ v).reshape(n, -1, D)
        first += n
    return out, lse


def exact(case, seed):
    if case["path"] == "tables":
        return None
    if case["path"] == "append":
        return _exact_append(case, seed)
    return _exact_attention(case, seed)
