"""The operators of the paged 8-bit key/value cache, in a plain form and as this
library's calls: what one serving step does between two sets of projections.

* ``plan``       block tables, slot map, positions and query offsets of a step,
                 from how many tokens each request holds and brings;
* ``append``     a step's keys and values into the cache, e4m3 with one scale
                 for each block of tokens and head;
* ``attention``  every token of the step against its request's cached keys and
                 values: single tokens, a few draft tokens, prompt chunks and
                 batches that mix them.

The cache: k [blocks, kv heads, block, D] and v [blocks, kv heads, D, block],
e4m3 codes as uint8, k_scale and v_scale fp32 [blocks, kv heads].

A case's lengths follow from the case alone (a low-discrepancy spread between
its bounds); the seed makes the values and the order of the blocks.
"""
import math

import torch

own = False  # set by who imports this: the library's calls instead of the plain form

DT = {"bf16": torch.bfloat16, "f16": torch.float16}
F8 = torch.float8_e4m3fn
MIN_EXP = -100  # the smallest scale is 2^-100


def listed():
    return [
        # One decode step of a small serving batch: 32 requests, a token each.
        {"name": "plan_decode", "op": "plan", "B": 32, "block": 16, "lo": 1, "hi": 4096, "new_lo": 1, "new_hi": 1,
         "ones": 0, "over": 0, "width": 512},
        # A large engine's step: most requests decode, the others bring prompts,
        # some have ended and give their blocks back.
        {"name": "plan_mixed", "op": "plan", "B": 1024, "block": 16, "lo": 0, "hi": 4000, "new_lo": 0, "new_hi": 512,
         "ones": 700, "over": 40, "width": 512},
        # The keys and values of that small batch's tokens.
        {"name": "append_decode", "op": "append", "dtype": "bf16", "B": 32, "Hkv": 8, "D": 128, "block": 16, "lo": 1,
         "hi": 2048, "new_lo": 1, "new_hi": 1, "ones": 0},
        # Eight prompts of about 2048 tokens, some behind a cached beginning that
        # ends inside a block.
        {"name": "append_prompts", "op": "append", "dtype": "bf16", "B": 8, "Hkv": 8, "D": 128, "block": 16, "lo": 0,
         "hi": 700, "new_lo": 1990, "new_hi": 2100, "ones": 0},
        # Ragged chunks at head dim 64 in fp16, as many kv heads as query heads,
        # long blocks.
        {"name": "append_chunks", "op": "append", "dtype": "f16", "B": 7, "Hkv": 12, "D": 64, "block": 64, "lo": 0,
         "hi": 1500, "new_lo": 37, "new_hi": 999, "ones": 0},
        # A single user's next token on a short context: latency.
        {"name": "attn_one", "op": "attention", "dtype": "bf16", "B": 1, "Hq": 32, "Hkv": 8, "D": 128, "block": 16,
         "lo": 777, "hi": 777, "q_lo": 1, "q_hi": 1, "ones": 0},
        # The small batch's tokens on ragged contexts.
        {"name": "attn_batch", "op": "attention", "dtype": "bf16", "B": 32, "Hq": 32, "Hkv": 8, "D": 128, "block": 16,
         "lo": 200, "hi": 4096, "q_lo": 1, "q_hi": 1, "ones": 0},
        # Two users with very long contexts: few rows, a long axis.
        {"name": "attn_long", "op": "attention", "dtype": "bf16", "B": 2, "Hq": 32, "Hkv": 8, "D": 128, "block": 64,
         "lo": 100001, "hi": 131072, "q_lo": 1, "q_hi": 1, "ones": 0},
        # A full batch of a model whose heads all have keys of their own: the
        # most cache read in a step.
        {"name": "attn_heads", "op": "attention", "dtype": "bf16", "B": 64, "Hq": 32, "Hkv": 32, "D": 128, "block": 32,
         "lo": 300, "hi": 6000, "q_lo": 1, "q_hi": 1, "ones": 0},
        # Verification of draft tokens: up to five tokens a request, head dim 64,
        # fp16.
        {"name": "attn_draft", "op": "attention", "dtype": "f16", "B": 16, "Hq": 16, "Hkv": 4, "D": 64, "block": 16,
         "lo": 333, "hi": 5000, "q_lo": 2, "q_hi": 5, "ones": 0},
        # Second chunks of four prompts: 2048 new tokens behind about as many.
        {"name": "attn_chunks", "op": "attention", "dtype": "bf16", "B": 4, "Hq": 32, "Hkv": 8, "D": 128, "block": 16,
         "lo": 3500, "hi": 4100, "q_lo": 2048, "q_hi": 2048, "ones": 0},
        # A step that mixes one prompt chunk into a decoding batch.
        {"name": "attn_mixed", "op": "attention", "dtype": "bf16", "B": 25, "Hq": 32, "Hkv": 8, "D": 128, "block": 16,
         "lo": 500, "hi": 6000, "q_lo": 511, "q_hi": 511, "ones": 24},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "append", "append", "attention", "attention", "attention", "attention"])
    block = rng.choice([16, 16, 32, 64, 128])
    if op == "plan":
        b = _log(rng, 1, 1024)
        hi = _log(rng, 16, 4000)
        new_hi = _log(rng, 1, 512)
        return {"op": op, "B": b, "block": block, "lo": rng.randint(0, hi), "hi": hi, "new_lo": rng.randint(0, new_hi),
                "new_hi": new_hi, "ones": rng.randint(0, b), "over": rng.randint(0, b // 8),
                "width": -(-(hi + new_hi) // block) + rng.randint(0, 300)}
    heads = rng.choice([(8, 1), (12, 12), (16, 4), (16, 16), (32, 8), (32, 8), (32, 32), (40, 8)])
    head = {"op": op, "dtype": rng.choice(["bf16", "bf16", "f16"])}
    if op == "append":
        d = rng.choice([64, 128])
        most = (1 << 24) // (heads[1] * d)  # tokens
        b = min(_log(rng, 1, 128), most)
        new_hi = max(1, _log(rng, 1, max(1, min(4096, most // b))))
        return dict(head, B=b, Hkv=heads[1], D=d, block=block, lo=0, hi=_log(rng, 1, 2048), new_lo=rng.randint(1, new_hi),
                    new_hi=new_hi, ones=rng.choice([0, 0, b // 2]))
    d = rng.choice([64, 128, 128])
    hi = _log(rng, 16, 65536)
    most = (1 << 29) // (hi * heads[1] * d)  # requests that keep the cache under 512 Mi keys and values
    q_hi = rng.choice([1, 1, 1, rng.randint(2, 8), _log(rng, 9, 2048)])
    q_hi = min(q_hi, hi, max(1, (1 << 28) // (hi * heads[0])))  # bounds the (row, key) pairs of a request
    b = max(1, min(_log(rng, 1, 64), most, (1 << 29) // (hi * heads[0] * q_hi)))
    return dict(head, B=b, Hq=heads[0], Hkv=heads[1], D=d, block=block, lo=rng.randint(q_hi, hi), hi=hi,
                q_lo=rng.randint(1, q_hi), q_hi=q_hi, ones=rng.choice([0, 0, b // 2]) if q_hi > 1 else 0)


# ---------------------------------------------------------------- lengths


def _spread(n, lo, hi, turn):
    """n whole numbers between lo and hi, dense at the short end."""
    f = [math.modf((i + 1) * turn)[0] for i in range(n)]
    return [lo + int((hi - lo) * x * x + 0.5) for x in f]


def _held(c):
    """Tokens in the cache before the step (plan, append)."""
    return _spread(c["B"], c["lo"], c["hi"], 0.6180339887498949)


def _brought(c):
    """Tokens each request brings (plan, append): `ones` of them a single one."""
    n = _spread(c["B"], c["new_lo"], c["new_hi"], 0.7548776662466927)
    return [1 if i < c["ones"] else x for i, x in enumerate(n)]


def _fresh(c):
    """What the plan is asked: tokens brought, -1 for a request that is over."""
    n = _brought(c)
    step = max(1, c["B"] // max(1, c["over"]))
    return [-1 if c["over"] and i % step == step - 1 and i // step < c["over"] else x for i, x in enumerate(n)]


def _attended(c):
    """(tokens in the cache, the step's own among them; tokens of the step) per request."""
    q = _spread(c["B"], c["q_lo"], c["q_hi"], 0.7548776662466927)
    q = [1 if i < c["ones"] else x for i, x in enumerate(q)]
    return [max(a, b) for a, b in zip(_spread(c["B"], c["lo"], c["hi"], 0.6180339887498949), q)], q


def _ceil(a, b):
    return -(-a // b)


# ---------------------------------------------------------------- inputs


def _gen(seed, k):
    return torch.Generator(device="cuda").manual_seed(1000 * (seed % (1 << 40)) + k)


def _randn(shape, seed, k):
    return torch.randn(shape, generator=_gen(seed, k), device="cuda")


def _perm(n, seed, k):
    return torch.randperm(n, generator=_gen(seed, k), device="cuda").to(torch.int32)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _tables(have, width, blocks, seed):
    """A table [B, width] whose first have[b] entries are blocks of their own in
    random order (the others 0), and the blocks left over."""
    ids = _perm(blocks, seed, 1)
    j = torch.arange(width, device="cuda", dtype=torch.int32)
    n = _ints(have)
    first = torch.cumsum(n, 0) - n
    at = (first[:, None] + j).clamp(max=blocks - 1).long()
    return torch.where(j < n[:, None], ids[at], 0).to(torch.int32).contiguous(), ids[sum(have):].clone()


def _two_to(e):
    """2^e in fp32, by its bits: exact."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _power(a):
    """The smallest power of two s with a <= 448 s, at least 2^-100."""
    m, e = torch.frexp(a)
    e = (e - 9 + (m > 0.875)).clamp(min=MIN_EXP)
    return _two_to(torch.where(a == 0, MIN_EXP, e))


def _codes(shape, dims, seed, k):
    """Codes and scales of a cache part: normal values, each channel with a
    strength of its own, as keys and values have."""
    blocks, heads = shape[:2]
    codes = torch.empty(shape, dtype=torch.uint8, device="cuda")
    scales = torch.empty((blocks, heads), device="cuda")
    strength = torch.exp(0.5 * _randn(dims, seed, k))
    step = max(1, (1 << 26) // (codes[0].numel()))
    for at in range(0, blocks, step):
        part = codes[at:at + step]
        x = _randn(part.shape, seed, k + 1 + at // step) * strength
        s = _power(x.abs().amax((2, 3)))
        part.copy_((x / s[..., None, None]).to(F8).view(torch.uint8))
        scales[at:at + step] = s
    return codes, scales


def _cache(c, blocks, seed):
    k, ks = _codes((blocks, c["Hkv"], c["block"], c["D"]), (c["D"],), seed, 100)
    v, vs = _codes((blocks, c["Hkv"], c["D"], c["block"]), (c["D"], 1), seed, 500000)
    return {"k": k, "v": v, "k_scale": ks, "v_scale": vs}


def _plan_inputs(c, seed):
    held, fresh = _held(c), _fresh(c)
    have = [_ceil(n, c["block"]) for n in held]
    need = [_ceil(h + max(0, f), c["block"]) - p for h, f, p in zip(held, fresh, have)]
    blocks = sum(have) + sum(need) + 8
    table, left = _tables(have, c["width"], blocks, seed)
    free = torch.zeros(blocks, dtype=torch.int32, device="cuda")
    free[:left.numel()] = left
    return {"cached": _ints(held), "fresh": _ints(fresh), "table": table, "free": free, "free_count": _ints([left.numel()]),
            "tokens": max(1, sum(max(0, f) for f in fresh))}


def _append_inputs(c, seed):
    held, new, bs = _held(c), _brought(c), c["block"]
    have = [_ceil(h + n, bs) for h, n in zip(held, new)]
    blocks = sum(have) + 4
    table, _ = _tables(have, max(have), blocks, seed)
    req = torch.repeat_interleave(torch.arange(c["B"], device="cuda"), _ints(new))
    first = torch.cumsum(_ints(new), 0) - _ints(new)
    pos = _ints(held)[req] + torch.arange(sum(new), device="cuda") - first[req]
    s = _cache(c, blocks, seed)
    shape, t = (sum(new), c["Hkv"], c["D"]), DT[c["dtype"]]
    # keys and values are parts of one projection's output [q | k | v]
    qkv = (_randn((shape[0], 3, c["Hkv"], c["D"]), seed, 2) * torch.exp(0.5 * _randn((c["D"],), seed, 3))).to(t)
    s.update(new_k=qkv[:, 1], new_v=qkv[:, 2], slots=(table[req, pos // bs] * bs + pos % bs).to(torch.int32),
             pages=torch.unique(table[req, pos // bs]).long())
    return s


def _attention_inputs(c, seed):
    lens, q = _attended(c)
    have = [_ceil(n, c["block"]) for n in lens]
    blocks = sum(have)
    s = _cache(c, blocks, seed)
    s["table"] = _tables(have, max(have), blocks, seed)[0]
    s["lens"] = _ints(lens)
    s["q_offsets"] = _ints([0] + [sum(q[:i + 1]) for i in range(len(q))])
    s["q"] = (_randn((sum(q), c["Hq"], c["D"]), seed, 2) * 0.6).to(DT[c["dtype"]])
    s.update(max_q=max(q), max_len=max(lens), scale=1.0 / math.sqrt(c["D"]))
    return s


def _inputs(case, seed):
    return {"plan": _plan_inputs, "append": _append_inputs, "attention": _attention_inputs}[case["op"]](case, seed)


def prepare(case, seed):
    c = dict(case)
    s = _inputs(c, seed)
    s["case"] = c
    i32 = dict(dtype=torch.int32, device="cuda")
    if c["op"] == "plan":
        b, t = c["B"], s["tokens"]
        s.update(lens=torch.empty(b, **i32), q_offsets=torch.empty(b + 1, **i32), slots=torch.empty(t, **i32),
                 positions=torch.empty(t, **i32), free_after=torch.empty(1, **i32))
    if c["op"] == "attention":
        s["o"] = torch.empty_like(s["q"])
    if own:  # the handle (pointers and sizes) and the workspace that a program keeps; no work on the data
        import pyc_amd
        if c["op"] != "plan":
            s["cache"] = pyc_amd.KvCache(s["k"], s["v"], s["k_scale"], s["v_scale"])
        if c["op"] == "attention":
            s["workspace"] = pyc_amd.kv_attention_workspace(c["B"], c["Hq"], c["Hkv"], c["D"], s["max_q"])
    return s


# ---------------------------------------------------------------- the plain forms


def _plan_plain(s):
    c, bs = s["case"], s["case"]["block"]
    cached, fresh, table, free, dev = s["cached"].long(), s["fresh"].long(), s["table"], s["free"], s["table"].device
    b, width, t = table.shape[0], table.shape[1], s["tokens"]
    n_free = s["free_count"].long()
    have = (cached + bs - 1) // bs
    over = fresh < 0
    # blocks of ended requests onto the stack, in request order
    back = torch.where(over, have, 0)
    end = torch.cumsum(back, 0)
    j = torch.arange(width, device=dev)
    put = n_free + (end - back)[:, None] + j
    put = torch.where(j < back[:, None], put, free.numel())
    stack = torch.cat([free, free.new_zeros(1)]).index_put((put.reshape(-1),), table.reshape(-1))
    top = n_free + end[-1]
    # what each request needs, and who gets it
    ask = torch.where(~over & (cached + fresh <= width * bs), fresh, 0)
    need = torch.where(ask > 0, (cached + ask + bs - 1) // bs - have, 0)
    blocks_end, tokens_end = torch.cumsum(need, 0), torch.cumsum(ask, 0)
    granted = (ask > 0) & ((need == 0) | (blocks_end <= top)) & (tokens_end <= t)
    need, ask = torch.where(granted, need, 0), torch.where(granted, ask, 0)
    blocks_end, tokens_end = torch.cumsum(need, 0), torch.cumsum(ask, 0)
    k = j - have[:, None]
    take = (top - 1 - (blocks_end - need)[:, None] - k).clamp(0, free.numel())
    s["table"].copy_(torch.where((k >= 0) & (k < need[:, None]), stack[take], table))
    free.copy_(stack[:-1])
    s["lens"].copy_(torch.where(over, 0, cached + ask))
    s["q_offsets"].copy_(torch.cat([tokens_end.new_zeros(1), tokens_end]))
    # a slot and a position for every token
    i = torch.arange(t, device=dev)
    r = torch.searchsorted(tokens_end, i, right=True).clamp(max=b - 1)
    pos = cached[r] + i - (tokens_end - ask)[r]
    slot = s["table"][r, (pos // bs).clamp(max=width - 1)] * bs + pos % bs
    live = i < tokens_end[-1]
    s["slots"].copy_(torch.where(live, slot, -1))
    s["positions"].copy_(torch.where(live, pos, -1))
    s["free_after"].copy_((top - blocks_end[-1]).reshape(1))


def _finite_max(x):
    return torch.where(torch.isfinite(x), x.abs(), 0).amax(-1)


def _append_part(x, codes, scales, slots, pages, bs, values):
    """One of k and v: `values` says that a block's tokens run along the last axis."""
    x = x.float()
    blk, off = (slots // bs).long(), (slots % bs).long()
    most = torch.zeros_like(scales).scatter_reduce_(0, blk[:, None].expand(-1, x.shape[1]), _finite_max(x), "amax")
    new = _power(most[pages])
    starts = torch.zeros(scales.shape[0], device=x.device).index_add_(0, blk, (off == 0).float())[pages] > 0
    old = scales[pages]
    s = torch.where(starts[:, None], new, torch.maximum(old, new))
    held = codes[pages].view(F8).float()
    shrunk = (held * (old / s)[..., None, None]).to(F8).view(torch.uint8)
    codes[pages] = torch.where((starts[:, None] | (s == old))[..., None, None], codes[pages], shrunk)
    scales[pages] = s
    q = torch.where(torch.isfinite(x), x * (1.0 / scales[blk])[..., None], math.nan).to(F8).view(torch.uint8)
    h = torch.arange(x.shape[1], device=x.device)
    if values:
        codes[blk[:, None], h, :, off[:, None]] = q
    else:
        codes[blk[:, None], h, off[:, None]] = q


def _append_plain(s):
    bs = s["case"]["block"]
    _append_part(s["new_k"], s["k"], s["k_scale"], s["slots"], s["pages"], bs, False)
    _append_part(s["new_v"], s["v"], s["v_scale"], s["slots"], s["pages"], bs, True)


def _attention_plain(s):
    c, q, lens, first = s["case"], s["q"], s["lens"], s["q_offsets"][:-1].long()
    b, hq, hk, d, bs, n = c["B"], c["Hq"], c["Hkv"], c["D"], c["block"], s["max_q"]
    pages = s["table"][:, :_ceil(s["max_len"], bs)].long()
    at = pages.shape[1] * bs
    k = s["k"][pages].view(F8).float() * s["k_scale"][pages][..., None, None]
    k = k.permute(0, 2, 4, 1, 3).reshape(b * hk, d, at)
    v = s["v"][pages].view(F8).float() * s["v_scale"][pages][..., None, None]
    v = v.permute(0, 2, 1, 4, 3).reshape(b * hk, at, d)
    # the requests' rows, padded to n tokens each
    i = torch.arange(n, device=q.device)
    count = s["q_offsets"][1:] - s["q_offsets"][:-1]
    row = torch.where(i < count[:, None], first[:, None] + i, q.shape[0])
    x = q[row.clamp(max=q.shape[0] - 1)].float() * s["scale"]
    x = x.reshape(b, n, hk, hq // hk, d).permute(0, 2, 1, 3, 4).reshape(b * hk, -1, d)
    p = torch.bmm(x, k).reshape(b, hk, n, hq // hk, at)
    last = (lens - count)[:, None] + i
    hidden = torch.arange(at, device=q.device) > last[..., None]
    p = p.masked_fill(hidden[:, None, :, None, :], -math.inf)
    p = torch.exp(p - p.amax(-1, keepdim=True))
    total = p.sum(-1, keepdim=True)
    o = torch.bmm(p.reshape(b * hk, -1, at), v).reshape(b, hk, n, hq // hk, d) / total
    o = o.permute(0, 2, 1, 3, 4).reshape(b * n, hq, d).to(q.dtype)
    out = q.new_empty((q.shape[0] + 1, hq, d)).index_put((row.reshape(-1),), o)
    s["o"].copy_(out[:-1])


def run(state):
    s, op = state, state["case"]["op"]
    if op == "plan":
        if own:
            import pyc_amd
            pyc_amd.kv_plan(s["cached"], s["fresh"], s["table"], s["free"], s["free_count"], s["case"]["block"], s["lens"],
                            s["q_offsets"], s["slots"], s["positions"], s["free_after"])
        else:
            _plan_plain(s)
        return {n: s[n] for n in ("table", "free", "lens", "q_offsets", "slots", "positions", "free_after")}
    if op == "append":
        if own:
            import pyc_amd
            pyc_amd.kv_append(s["new_k"], s["new_v"], s["slots"], s["cache"])
        else:
            _append_plain(s)
        return {"k": s["k"].view(F8), "v": s["v"].view(F8), "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    if own:
        import pyc_amd
        pyc_amd.kv_attention(s["q"], s["cache"], s["table"], s["lens"], s["q_offsets"], s["o"], s["scale"], s["max_q"],
                             max_len=s["max_len"], workspace=s["workspace"])
    else:
        _attention_plain(s)
    return {"o": s["o"]}


# ---------------------------------------------------------------- measures


def work(case):
    c = case
    if c["op"] == "plan":
        held, fresh, bs = _held(c), _fresh(c), c["block"]
        tokens = sum(max(0, f) for f in fresh)
        read = sum(_ceil(h + f, bs) - h // bs for h, f in zip(held, fresh) if f > 0)  # table entries of the slots
        back = sum(_ceil(h, bs) for h, f in zip(held, fresh) if f < 0)
        new = sum(_ceil(h + f, bs) - _ceil(h, bs) for h, f in zip(held, fresh) if f > 0)
        return {"bytes": 4 * (4 * c["B"] + 3 + 2 * tokens + read + 2 * back + 2 * new), "flops": 0}
    if c["op"] == "append":
        n = sum(_brought(c))
        pages = sum(_ceil(h + m, c["block"]) - h // c["block"] for h, m in zip(_held(c), _brought(c)))
        return {"bytes": n * (2 * c["Hkv"] * c["D"] * (2 + 1) + 4) + 16 * pages * c["Hkv"], "flops": 4 * n * c["Hkv"] * c["D"]}
    lens, q = _attended(c)
    pairs = sum(m * (n - m) + m * (m + 1) // 2 for n, m in zip(lens, q))
    pages = sum(_ceil(n, c["block"]) for n in lens)
    return {"bytes": 2 * sum(lens) * c["Hkv"] * c["D"] + 4 * sum(q) * c["Hq"] * c["D"] + pages * (4 + 8 * c["Hkv"]),
            "flops": 4 * pairs * c["Hq"] * c["D"]}


def _round_e4m3(x):
    """x, |x| <= 448, to the nearest value with three mantissa bits and no
    exponent below -6, ties to even."""
    e = torch.frexp(x)[1].clamp(min=-5) - 1
    step = _two_to(e - 3).double()
    return torch.round(x / step) * step


def _plan_exact(c, x):
    bs, width = c["block"], c["width"]
    cached, fresh, table = x["cached"].tolist(), x["fresh"].tolist(), x["table"].cpu()
    free, stack = x["free"].cpu(), x["free"].tolist()[:int(x["free_count"])]
    for b, f in enumerate(fresh):
        if f < 0:
            stack += table[b, :_ceil(cached[b], bs)].tolist()
    free[:len(stack)] = torch.tensor(stack, dtype=torch.int32)
    lens, offsets, slots, positions = [], [0], [], []
    for b, f in enumerate(fresh):  # the inputs ask for no more than there is: everybody is served
        had, n = cached[b], max(0, f)
        for j in range(_ceil(had, bs), _ceil(had + n, bs)):
            table[b, j] = stack.pop()
        lens.append(0 if f < 0 else had + n)
        offsets.append(offsets[-1] + n)
        pos = list(range(had, had + n))
        positions += pos
        slots += [int(table[b, p // bs]) * bs + p % bs for p in pos]
    rest = [-1] * (x["tokens"] - len(slots))
    i32 = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    return {"table": table, "free": free, "lens": i32(lens), "q_offsets": i32(offsets), "slots": i32(slots + rest),
            "positions": i32(positions + rest), "free_after": i32([len(stack)])}


def _append_exact(c, x):
    bs, blk = c["block"], (x["slots"] // c["block"]).long()
    off = (x["slots"] % bs).long()
    out = {}
    for name in ("k", "v"):
        codes, old = x[name].view(F8).double(), x[name + "_scale"].double()
        if name == "v":
            codes = codes.transpose(2, 3).contiguous()
        rows = x["new_" + name].double()
        most = torch.zeros_like(old).scatter_reduce_(0, blk[:, None].expand(-1, old.shape[1]), rows.abs().amax(-1), "amax")
        new = _two_to(torch.ceil(torch.log2(most / 448.0)).clamp(min=MIN_EXP)).double()
        touched = torch.zeros(old.shape[0], dtype=torch.bool, device=old.device)
        touched[blk] = True
        starts = torch.zeros_like(touched)
        starts[blk[off == 0]] = True
        s = torch.where(touched[:, None], torch.where(starts[:, None], new, torch.maximum(old, new)), old)
        grown = touched & ~starts
        codes[grown] = _round_e4m3(codes[grown] * (old / s)[grown][..., None, None])
        codes[blk, :, off] = _round_e4m3(rows / s[blk][..., None])
        out[name] = codes.transpose(2, 3).contiguous() if name == "v" else codes
        out[name + "_scale"] = s
    return out


def _attention_exact(c, x):
    lens, q = _attended(c)
    g, bs, out, at = c["Hq"] // c["Hkv"], c["block"], [], 0
    for b, (n, m) in enumerate(zip(lens, q)):
        ids = x["table"][b, :_ceil(n, bs)].long()
        k = (x["k"][ids].view(F8).double() * x["k_scale"][ids].double()[..., None, None]).transpose(0, 1)
        v = (x["v"][ids].view(F8).double() * x["v_scale"][ids].double()[..., None, None]).permute(1, 0, 3, 2)
        k, v = (t.reshape(c["Hkv"], -1, c["D"])[:, :n] for t in (k, v))
        rows = x["q"][at:at + m].double()
        hidden = torch.arange(n, device=k.device)[None, :] > torch.arange(n - m, n, device=k.device)[:, None]
        o = torch.empty_like(rows)
        for h in range(c["Hkv"]):
            s = (rows[:, h * g:(h + 1) * g].reshape(m * g, -1) @ k[h].t().contiguous()).reshape(m, g, n) * x["scale"]
            p = torch.softmax(s.masked_fill(hidden[:, None], -math.inf), -1)
            o[:, h * g:(h + 1) * g] = (p.reshape(m * g, n) @ v[h].contiguous()).reshape(m, g, -1)
        out.append(o)
        at += m
    return {"o": torch.cat(out)}


def exact(case, seed):
    x = _inputs(dict(case), seed)
    return {"plan": _plan_exact, "append": _append_exact, "attention": _attention_exact}[case["op"]](case, x)
