"""The paged 8-bit key/value cache's operators restated plainly, in 64 bits on
the CPU, and inputs for their tests."""
import math

import numpy as np
import torch

F8 = torch.float8_e4m3fn
DT = {"bf16": torch.bfloat16, "f16": torch.float16}
HALF = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}  # half a step of the type, relative


def ceil_div(a, b):
    return -(-a // b)


# ---------------------------------------------------------------- plan


def plan_ref(cached, fresh, table, free, count, bs, tokens):
    """One request after the other, with Python integers."""
    table, free = table.copy(), free.copy()
    width, cap = table.shape[1], len(free)
    cached = [min(max(int(c), 0), width * bs) for c in cached]
    top = min(max(count, 0), cap)
    for b, f in enumerate(fresh):
        if f < 0:
            for j in range(ceil_div(cached[b], bs)):
                if top < cap:
                    free[top] = table[b, j]
                    top += 1
    lens, offsets, slots, pos = [], [0], [], []
    asked_blocks = asked_tokens = 0
    left = top
    for b, f in enumerate(fresh):
        f = int(f)
        have, n = ceil_div(cached[b], bs), 0
        if f > 0 and cached[b] + f <= width * bs:
            need = ceil_div(cached[b] + f, bs) - have
            asked_blocks += need
            asked_tokens += f
            if (need == 0 or asked_blocks <= top) and asked_tokens <= tokens:
                n = f
                for j in range(need):
                    left -= 1
                    table[b, have + j] = free[left]
        lens.append(0 if f < 0 else cached[b] + n)
        offsets.append(offsets[-1] + n)
        for p in range(cached[b], cached[b] + n):
            pos.append(p)
            slots.append(int(table[b, p // bs]) * bs + p % bs)
    rest = [-1] * (tokens - len(slots))
    i32 = lambda v: np.array(v, np.int32)  # noqa: E731
    return {"table": table, "free": free, "lens": i32(lens), "q_offsets": i32(offsets), "slots": i32(slots + rest),
            "positions": i32(pos + rest), "free_after": i32([left])}


# ---------------------------------------------------------------- cache


def round_e4m3(x):
    """float64 to the nearest e4m3 value, ties to even; not finite -> NaN."""
    ok = torch.isfinite(x)
    y = torch.where(ok, x, 0.0)
    e = torch.clamp(torch.frexp(y)[1] - 1, min=-6)
    step = torch.ldexp(torch.ones_like(y), e - 3)
    return torch.where(ok, torch.round(y / step) * step, math.nan)


def power_scale(a):
    """The smallest power of two s >= 2^-100 with a <= 448 s."""
    s = 2.0 ** -100
    while a > 448.0 * s:
        s *= 2.0
    return s


def append_ref(cache, k, v, slots):
    """cache: dict of k, v (float64 code values, [N,H,bs,D] and [N,H,D,bs]) and
    k_scale, v_scale (float64). In place."""
    bs = cache["k"].shape[2]
    blocks = {}
    for t, s in enumerate(slots):
        if 0 <= s < cache["k"].shape[0] * bs:
            blocks.setdefault(s // bs, []).append((t, s % bs))
    for name, x in (("k", k.double()), ("v", v.double())):
        codes = cache[name] if name == "k" else cache[name].transpose(2, 3)
        for blk, rows in blocks.items():
            for h in range(x.shape[1]):
                new = x[[t for t, _ in rows], h]
                s_new = power_scale(float(torch.where(torch.isfinite(new), new.abs(), 0.0).max()))
                old = float(cache[name + "_scale"][blk, h])
                s = s_new
                if all(o != 0 for _, o in rows) and math.isfinite(old) and old > 0:
                    s = max(old, s_new)
                    if s > old:
                        codes[blk, h] = round_e4m3(codes[blk, h] * (old / s))
                cache[name + "_scale"][blk, h] = s
                for (_, o), row in zip(rows, new):
                    codes[blk, h, o] = round_e4m3(row / s)


def random_cache(blocks, heads, bs, d, seed, scale_spread=2):
    """Codes of normal values, scales powers of two around 2^-7 (and one odd
    scale), on the CPU: dict of uint8 codes and fp32 scales."""
    g = torch.Generator().manual_seed(seed)
    out = {}
    for name, shape in (("k", (blocks, heads, bs, d)), ("v", (blocks, heads, d, bs))):
        x = torch.randn(shape, generator=g) * 100.0
        out[name] = x.clamp(-448, 448).to(F8).view(torch.uint8)
        e = torch.randint(-scale_spread, scale_spread + 1, (blocks, heads), generator=g).float()
        out[name + "_scale"] = torch.pow(2.0, e - 7.0)
    out["k_scale"][0, 0] = 0.0123
    out["v_scale"][0, 0] = 0.0077
    return out


def values(cache):
    """The cache's codes as float64 and its scales as float64."""
    return {"k": cache["k"].view(F8).double(), "v": cache["v"].view(F8).double(),
            "k_scale": cache["k_scale"].double(), "v_scale": cache["v_scale"].double()}


# ---------------------------------------------------------------- attention


def attention_ref(q, cache, table, lens, offsets, scale, max_q=1 << 30, out=None, only=None):
    """(o, bound, computed): float64 outputs; per output, how far a result of the
    types used may be off but for the output's own rounding; which rows of q the
    call computes. only: the tokens that are looked at (the others are not `computed`).

    With a_j = |v_j| and P = softmax: o = sum P v. The kernel's scores are off by
    at most ds = (D + 4) 2^-24 S (S = sum_d |q_d k_jd| scale, largest over j; fp32
    products of D terms, the scales' products, one subtraction), so P by a factor
    e^(2 ds); sums over n keys by n 2^-24 each for numerator and denominator, and a
    2^-22 for the exponential; P rounded to 16 bits by `half`. All scale A = sum P
    |v|."""
    hq, d = q.shape[1], q.shape[2]
    hk, bs = cache["k"].shape[1], cache["k"].shape[2]
    g, width, nb = hq // hk, table.shape[1], cache["k"].shape[0]
    half = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -15}[q.dtype]
    c = values(cache)
    o = torch.zeros(q.shape, dtype=torch.float64) if out is None else out.double().clone()
    bound = torch.zeros(q.shape, dtype=torch.float64)
    done = torch.zeros(q.shape[0], dtype=torch.bool)
    x = q.double()
    for b in range(len(lens)):
        n_keys = min(max(int(lens[b]), 0), width * bs)
        first, end = int(offsets[b]), int(offsets[b + 1])
        ids = [int(table[b, j]) for j in range(ceil_div(n_keys, bs))]
        there = torch.tensor([0 <= i < nb for i in ids], dtype=torch.bool).repeat_interleave(bs)[:n_keys]
        ids = torch.tensor([i if 0 <= i < nb else 0 for i in ids], dtype=torch.long)
        k = (c["k"][ids] * c["k_scale"][ids][..., None, None]).transpose(0, 1).reshape(hk, -1, d)[:, :n_keys]
        v = (c["v"][ids] * c["v_scale"][ids][..., None, None]).permute(1, 0, 3, 2).reshape(hk, -1, d)[:, :n_keys]
        for i in range(min(end - first, max_q)):
            t = first + i
            if only is not None and t not in only:
                continue
            done[t] = True
            see = max(0, min(n_keys, n_keys - (end - first) + i + 1))
            keep = there[:see]
            if see == 0 or not bool(keep.any()):
                o[t] = 0.0
                continue
            for h in range(hq):
                kk, vv = k[h // g, :see][keep], v[h // g, :see][keep]
                s = kk @ x[t, h] * scale
                p = torch.softmax(s, 0)
                o[t, h] = p @ vv
                big = float((kk.abs() @ x[t, h].abs()).max()) * abs(scale)
                rel = half + 2 * (d + 4) * 2.0 ** -24 * big + 2 * see * 2.0 ** -24 + 2.0 ** -21
                bound[t, h] = rel * (p @ vv.abs())
    return o, bound, done
