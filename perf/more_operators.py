"""The operators of a feed-forward layer of experts and of 4-bit weights, in a
plain form and as this library's calls: what one layer of such a model does
between two attentions.

* ``route``    each token's k experts and their weights from the router's
               logits, and the order that puts the tokens of one expert together;
* ``grouped``  the rows of every expert times that expert's 16-bit weights, with
               the gather of the rows before it and the gate behind it;
* ``w4``       the same with weights of 4 bits and a scale for each group along
               the row, for a dense layer (one expert that has every row) or many;
* ``combine``  each token's weighted sum of its experts' rows.

Weights are [experts, N, K]; 4-bit codes [experts, N, K / 2] uint8 with the even k
in the low half of a byte, scales [experts, N, K / group] of the rows' type and, in
some cases, zero points [experts, N, K / group] uint8 (8 without): a weight is
(code - zero) * scale. A gated product has N = 2 F rows of weights, F gates and
then F values, and F columns: silu(gate) * value.

How many rows each expert has follows from the case alone; the seed makes the
values, which tokens and which experts.
"""
import math

import numpy as np
import torch

own = False  # set by who imports this: the library's calls instead of the plain form

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # The router of a small decoding batch: latency.
        {"name": "route_decode", "op": "route", "dtype": "f32", "T": 32, "E": 64, "k": 8, "normalize": True, "pad": 0},
        # A prompt's tokens, the last ones padding whose logits are -infinity.
        {"name": "route_prompt", "op": "route", "dtype": "bf16", "T": 8200, "E": 128, "k": 8, "normalize": False,
         "pad": 8},
        # A single user's next token through four small experts: latency and the
        # stream of their weights.
        {"name": "grouped_token", "op": "grouped", "dtype": "bf16", "T": 1, "k": 4, "E": 32, "K": 2048, "N": 2048,
         "epi": "gate", "bias": False, "gather": True},
        # A decoding batch: every expert has a few rows, all weights are read.
        {"name": "grouped_decode", "op": "grouped", "dtype": "bf16", "T": 32, "k": 8, "E": 64, "K": 2048, "N": 2816,
         "epi": "gate", "bias": False, "gather": True},
        # The second product of a chunk of prompts in fp16: rows already in the
        # experts' order, a width that is no multiple of a tile, skewed experts.
        {"name": "grouped_chunk", "op": "grouped", "dtype": "f16", "T": 700, "k": 8, "E": 64, "K": 1408, "N": 2040,
         "epi": "none", "bias": False, "gather": False},
        # A long prompt through a few large experts: bound by the matrix units.
        {"name": "grouped_prompt", "op": "grouped", "dtype": "bf16", "T": 4096, "k": 2, "E": 8, "K": 4096, "N": 22016,
         "epi": "gate", "bias": False, "gather": True},
        # A single user's next token through one 4-bit layer.
        {"name": "w4_token", "op": "w4", "dtype": "bf16", "T": 1, "k": 1, "E": 1, "K": 4096, "N": 11008, "group": 128,
         "zeros": False, "epi": "none", "bias": False, "gather": False},
        # A batch of tokens in fp16, short groups with zero points, a deep row.
        {"name": "w4_batch", "op": "w4", "dtype": "f16", "T": 23, "k": 1, "E": 1, "K": 11008, "N": 4096, "group": 32,
         "zeros": True, "epi": "none", "bias": True, "gather": False},
        # A decoding batch through 4-bit experts.
        {"name": "w4_experts", "op": "w4", "dtype": "bf16", "T": 16, "k": 4, "E": 32, "K": 4096, "N": 2816,
         "group": 64, "zeros": False, "epi": "gate", "bias": False, "gather": True},
        # A prompt through a 4-bit layer.
        {"name": "w4_prompt", "op": "w4", "dtype": "bf16", "T": 1999, "k": 1, "E": 1, "K": 4096, "N": 11008,
         "group": 128, "zeros": False, "epi": "relu", "bias": False, "gather": False},
        # A decoding batch's experts summed onto the residual stream.
        {"name": "combine_decode", "op": "combine", "dtype": "bf16", "T": 32, "k": 8, "E": 64, "H": 2048, "base": True},
        # A prompt's.
        {"name": "combine_prompt", "op": "combine", "dtype": "bf16", "T": 8200, "k": 8, "E": 128, "H": 2048,
         "base": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["route", "grouped", "grouped", "grouped", "w4", "w4", "w4", "combine"])
    half = rng.choice(["bf16", "bf16", "f16"])
    experts = _log(rng, 2, 256)
    k = rng.randint(1, min(8, experts))
    if op == "route":
        t = _log(rng, 1, 16384)
        return {"op": op, "dtype": rng.choice(["f32", "bf16", "f16"]), "T": t, "E": experts, "k": k,
                "normalize": rng.choice([True, False]), "pad": rng.choice([0, 0, t // 10])}
    if op == "combine":
        h = rng.choice([_log(rng, 64, 8192), 8 * _log(rng, 8, 1024)])
        return {"op": op, "dtype": half, "T": max(1, min(_log(rng, 1, 16384), (1 << 27) // (k * h))), "k": k, "E": experts,
                "H": h, "base": rng.choice([True, False])}
    epi = rng.choice(["none", "relu", "gate", "gate"])
    t = _log(rng, 1, 4096)
    if op == "w4":
        group = rng.choice([32, 64, 128])
        depth = group * max(1, _log(rng, 256, 11008) // group)
        if rng.random() < 0.5:
            experts = k = 1
    else:
        depth = rng.choice([8 * _log(rng, 8, 1376), 64 * _log(rng, 1, 172), 64 * _log(rng, 1, 172), _log(rng, 64, 4096)])
    n = rng.choice([8 * _log(rng, 8, 1376), 128 * _log(rng, 1, 86), _log(rng, 64, 4096)])
    if epi == "gate":
        n *= 2
    most = (1 << 29) // (n * depth)  # experts that keep the weights under 512 Mi
    experts = max(1, min(experts, most))
    k = min(k, experts)
    t = max(1, min(t, int(7e11) // (k * n * depth)))
    c = {"op": op, "dtype": half, "T": t, "k": k, "E": experts, "K": depth, "N": n, "epi": epi,
         "bias": rng.choice([False, False, True]), "gather": k > 1 and rng.random() < 0.5}
    return dict(c, group=group, zeros=rng.choice([True, False])) if op == "w4" else c


# ---------------------------------------------------------------- inputs


def _gen(seed, k):
    return torch.Generator(device="cuda").manual_seed(1000 * (seed % (1 << 40)) + k)


def _randn(shape, seed, k):
    return torch.randn(shape, generator=_gen(seed, k), device="cuda")


def _normal(shape, factor, dtype, seed, k):
    """Normal values times factor, made in pieces along the first axis."""
    out = torch.empty(shape, dtype=dtype, device="cuda")
    for i in range(shape[0]):
        out[i] = _randn(shape[1:], seed, k + i) * factor
    return out


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _choices(c):
    """[T, k] experts before they are renamed: a token takes k neighbours, most
    tokens among the first ones."""
    u = np.modf((np.arange(c["T"]) + 1) * 0.6180339887498949)[0]
    return ((c["E"] * u * u).astype(np.int64)[:, None] + np.arange(c["k"])) % c["E"]


def _active(c):
    return int(np.unique(_choices(c)).size)


def _order(c, seed):
    """(rows of each expert, the flat (token, place) indexes in the experts' order)."""
    r = np.random.default_rng(seed % (1 << 40))
    flat = r.permutation(c["E"])[_choices(c)[r.permutation(c["T"])]].reshape(-1)
    return np.bincount(flat, minlength=c["E"]).tolist(), np.argsort(flat, kind="stable")


def _ends(counts):
    return _ints([0] + np.cumsum(counts).tolist())


def _route_inputs(c, seed):
    x = _randn((c["T"], c["E"]), seed, 1) * 1.5 + _randn((c["E"],), seed, 2) * 0.5
    if c["pad"]:
        x[c["T"] - c["pad"]:] = -math.inf
    return {"logits": x.to(DT[c["dtype"]])}


def _product_inputs(c, seed):
    t, counts, order = DT[c["dtype"]], *_order(c, seed)
    p = c["T"] * c["k"]
    strength = torch.exp(0.5 * _randn((c["K"],), seed, 1))
    s = {"x": (_randn((c["T"] if c["gather"] else p, c["K"]), seed, 2) * strength).to(t), "counts": counts,
         "offsets": _ends(counts), "rows": _ints(order.tolist()) if c["gather"] else None, "bias": None}
    if c["bias"]:
        s["bias"] = 0.1 * _randn((c["E"], c["N"]), seed, 3)
    shape, size = (c["E"], c["N"], c["K"]), 1.0 / math.sqrt(c["K"])
    if c["op"] == "grouped":
        return dict(s, w=_normal(shape, size, t, seed, 100))
    # codes of weights whose groups have about this spread
    lo = torch.empty((c["E"], c["N"], c["K"] // 2), dtype=torch.uint8, device="cuda")
    for e in range(c["E"]):
        q = (_randn(shape[1:], seed, 100 + e) * 2.7 + 8.0).round_().clamp_(0, 15).to(torch.uint8)
        lo[e] = q[:, 0::2] | (q[:, 1::2] << 4)
    g = (c["E"], c["N"], c["K"] // c["group"])
    s.update(w=lo, scale=(torch.exp(0.3 * _randn(g, seed, 4)) * (size / 2.7)).to(t), zeros=None)
    if c["zeros"]:
        s["zeros"] = torch.randint(5, 11, g, generator=_gen(seed, 5), device="cuda", dtype=torch.uint8)
    return s


def _combine_inputs(c, seed):
    counts, order = _order(c, seed)
    p, t = c["T"] * c["k"], DT[c["dtype"]]
    places = np.empty(p, np.int32)
    places[order] = np.arange(p)
    w = torch.softmax(_randn((c["T"], c["k"]), seed, 1), -1)
    return {"y": _randn((p, c["H"]), seed, 2).to(t), "weights": w, "places": _ints(places.tolist()),
            "base": _randn((c["T"], c["H"]), seed, 3).to(t) if c["base"] else None}


def _inputs(case, seed):
    return {"route": _route_inputs, "grouped": _product_inputs, "w4": _product_inputs,
            "combine": _combine_inputs}[case["op"]](case, seed)


def prepare(case, seed):
    c = dict(case)
    s = _inputs(c, seed)
    s["case"] = c
    if c["op"] == "route":
        n, i32 = c["T"] * c["k"], dict(dtype=torch.int32, device="cuda")
        s.update(ids=torch.empty((c["T"], c["k"]), **i32), weights=torch.empty((c["T"], c["k"]), device="cuda"),
                 offsets=torch.empty(c["E"] + 1, **i32), rows=torch.empty(n, **i32), places=torch.empty(n, **i32))
        if own:
            import pyc_amd
            s["workspace"] = pyc_amd.moe_route_workspace(c["T"], c["E"], c["k"])
    elif c["op"] == "combine":
        s["out"] = torch.empty((c["T"], c["H"]), dtype=s["y"].dtype, device="cuda")
    else:
        n = c["N"] // 2 if c["epi"] == "gate" else c["N"]
        s["y"] = torch.empty((c["T"] * c["k"], n), dtype=s["x"].dtype, device="cuda")
    return s


# ---------------------------------------------------------------- the plain forms


def _route_plain(s):
    k, x = s["ids"].shape[1], s["logits"].float()
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    order = torch.sort(x, dim=-1, descending=True, stable=True)[1][:, :k]
    chosen = torch.gather(p, 1, order)
    there = torch.gather(x, 1, order) > -math.inf
    total = (chosen if s["case"]["normalize"] else p).sum(-1, keepdim=True)
    s["weights"].copy_(torch.where(there, chosen / torch.where(total == 0, 1.0, total), 0.0))
    s["ids"].copy_(torch.where(there, order, -1))
    # the flat places in the order of their experts, the ones without an expert last
    experts = x.shape[1]
    flat = torch.where(there, order, experts).reshape(-1)
    by = torch.sort(flat, stable=True)[1]
    count = torch.zeros(experts + 1, dtype=torch.int64, device=x.device).index_add_(0, flat, torch.ones_like(flat))
    s["offsets"].copy_(torch.cumsum(count, 0) - count)
    at = torch.arange(flat.numel(), device=x.device)
    s["rows"].copy_(torch.where(at < s["offsets"][-1], by, -1))
    s["places"].copy_(torch.where(flat < experts, torch.empty_like(at).index_copy_(0, by, at), -1))


def _weights(s, e):
    if s["case"]["op"] == "grouped":
        return s["w"][e].float()
    q, g = s["w"][e], s["case"]["group"]
    q = torch.stack([q & 15, q >> 4], -1).reshape(q.shape[0], -1, g).float()
    q = q - (8.0 if s["zeros"] is None else s["zeros"][e].float()[..., None])
    return (q * s["scale"][e].float()[..., None]).reshape(q.shape[0], -1)


def _product_plain(s):
    c, at = s["case"], 0
    for e, n in enumerate(s["counts"]):
        if n == 0:
            continue
        x = s["x"][s["rows"][at:at + n] // c["k"]] if c["gather"] else s["x"][at:at + n]
        h = x.float() @ _weights(s, e).t()
        if s["bias"] is not None:
            h = h + s["bias"][e]
        if c["epi"] == "relu":
            h = torch.clamp(h, min=0.0)
        if c["epi"] == "gate":
            a, b = h[:, :c["N"] // 2], h[:, c["N"] // 2:]
            h = a / (1.0 + torch.exp(-a)) * b
        s["y"][at:at + n] = h.to(s["y"].dtype)
        at += n


def _combine_plain(s):
    t, k = s["weights"].shape
    y = s["y"][s["places"].long()].reshape(t, k, -1).float()
    o = (y * s["weights"][..., None]).sum(1)
    if s["base"] is not None:
        o = o + s["base"].float()
    s["out"].copy_(o)


EPILOGUE = {"none": 0, "relu": 2, "gate": 4}


def run(state):
    s, c = state, state["case"]
    if own:
        import pyc_amd
    if c["op"] == "route":
        if own:
            pyc_amd.moe_route(s["logits"], s["ids"], s["weights"], s["offsets"], s["rows"], s["places"],
                              normalize=c["normalize"], workspace=s["workspace"])
        else:
            _route_plain(s)
        return {n: s[n] for n in ("ids", "weights", "offsets", "rows", "places")}
    if c["op"] == "combine":
        if own:
            pyc_amd.moe_combine(s["y"], s["weights"], s["places"], s["out"], base=s["base"])
        else:
            _combine_plain(s)
        return {"out": s["out"]}
    if not own:
        _product_plain(s)
    elif c["op"] == "grouped":
        pyc_amd.grouped_gemm(s["x"], s["w"], s["offsets"], s["y"], rows=s["rows"], fan=c["k"], bias=s["bias"],
                             epilogue=EPILOGUE[c["epi"]])
    elif c["E"] == 1:
        one = lambda v: None if v is None else v[0]  # noqa: E731
        pyc_amd.w4a16_gemm(s["x"], s["w"][0], s["scale"][0], s["y"], zeros=one(s["zeros"]), bias=one(s["bias"]),
                           epilogue=EPILOGUE[c["epi"]])
    else:
        pyc_amd.w4a16_grouped_gemm(s["x"], s["w"], s["scale"], s["offsets"], s["y"], zeros=s["zeros"], rows=s["rows"],
                                   fan=c["k"], bias=s["bias"], epilogue=EPILOGUE[c["epi"]])
    return {"y": s["y"]}


# ---------------------------------------------------------------- measures


def work(case):
    c, size = case, {"bf16": 2, "f16": 2, "f32": 4}[case["dtype"]]
    p = c["T"] * c["k"]
    if c["op"] == "route":
        return {"bytes": c["T"] * c["E"] * size + 16 * p + 4 * (c["E"] + 1), "flops": 0}
    if c["op"] == "combine":
        return {"bytes": size * c["H"] * (p + c["T"] * (2 if c["base"] else 1)) + 8 * p, "flops": 2 * p * c["H"]}
    weights = c["N"] * c["K"] * 2
    if c["op"] == "w4":
        weights = c["N"] * (c["K"] // 2 + c["K"] // c["group"] * (3 if c["zeros"] else 2))
    if c["bias"]:
        weights += 4 * c["N"]
    n = c["N"] // 2 if c["epi"] == "gate" else c["N"]
    rows = c["T"] if c["gather"] else p
    return {"bytes": weights * _active(c) + 2 * (rows * c["K"] + p * n) + 4 * (p * c["gather"] + c["E"] + 1),
            "flops": 2 * p * c["N"] * c["K"]}


def _route_exact(c, x):
    l, n = x["logits"].double().cpu().numpy(), c["T"] * c["k"]
    ids, w = np.full((c["T"], c["k"]), -1, np.int32), np.zeros((c["T"], c["k"]))
    for t, row in enumerate(l):
        top = row.max()
        if top == -math.inf:
            continue
        p = np.exp(row - top)
        best = np.lexsort((np.arange(c["E"]), -row))[:c["k"]]  # larger first, then the lower index
        best = best[row[best] > -math.inf]
        ids[t, :len(best)] = best
        w[t, :len(best)] = p[best] / (p[best].sum() if c["normalize"] else p.sum())
    rows, places, offsets = np.full(n, -1, np.int32), np.full(n, -1, np.int32), [0]
    for e in range(c["E"]):
        f = np.nonzero(ids.reshape(-1) == e)[0]
        rows[offsets[-1]:offsets[-1] + len(f)] = f
        places[f] = offsets[-1] + np.arange(len(f))
        offsets.append(offsets[-1] + len(f))
    return {"ids": torch.from_numpy(ids), "weights": torch.from_numpy(w), "offsets": torch.tensor(offsets, dtype=torch.int32),
            "rows": torch.from_numpy(rows), "places": torch.from_numpy(places)}


def _product_exact(c, x):
    ends, k, out = x["offsets"].tolist(), c["K"], []
    step = max(1, (1 << 27) // k)
    for e in range(c["E"]):
        a, b = ends[e], ends[e + 1]
        if a == b:
            continue
        src = torch.arange(a, b, device="cuda")
        if c["gather"]:
            src = torch.div(x["rows"][a:b].long(), c["k"], rounding_mode="floor")
        rows, parts = x["x"].double().index_select(0, src), []
        for n in range(0, c["N"], step):
            w = x["w"][e, n:n + step]
            if c["op"] == "w4":
                codes = torch.empty((w.shape[0], k), dtype=torch.float64, device="cuda")
                codes[:, 0::2], codes[:, 1::2] = w % 16, w // 16
                shape = (w.shape[0], k // c["group"], c["group"])
                zero = 8 if x["zeros"] is None else x["zeros"][e, n:n + step].double().unsqueeze(-1)
                w = ((codes.view(shape) - zero) * x["scale"][e, n:n + step].double().unsqueeze(-1)).view(-1, k)
            parts.append(torch.mm(rows, w.double().t()))
        h = torch.cat(parts, 1)
        if x["bias"] is not None:
            h += x["bias"][e].double()
        if c["epi"] == "relu":
            h = torch.maximum(h, torch.zeros_like(h))
        elif c["epi"] == "gate":
            gate, value = h.chunk(2, 1)
            h = gate * torch.sigmoid(gate) * value
        out.append(h)
    return {"y": torch.cat(out)}


def _combine_exact(c, x):
    o = x["base"].double() if c["base"] else torch.zeros((c["T"], c["H"]), dtype=torch.float64, device="cuda")
    at = x["places"].long().view(c["T"], c["k"])
    for j in range(c["k"]):
        o += x["weights"][:, j:j + 1].double() * x["y"][at[:, j]].double()
    return {"out": o}


def exact(case, seed):
    c = dict(case)
    x = _inputs(c, seed)
    return {"route": _route_exact, "grouped": _product_exact, "w4": _product_exact, "combine": _combine_exact}[c["op"]](c, x)
