"""The operators of a layer of experts and of 4-bit weights restated plainly, in
64 bits on the CPU, inputs for their tests, and how far results may be off."""
import ctypes
import math

import numpy as np
import torch

import pyc_amd

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # half a step of the type, relative
TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}  # half the smallest step
MOST = {torch.bfloat16: math.inf, torch.float16: 65520.0}  # from here on a value rounds to infinity (bf16: past any here)
U = 2.0 ** -24  # half a step of fp32, relative
GATE, RELU = 4, 2


def rounded(h, d, dtype):
    """How far h, off by at most d, may be off once rounded to dtype: by half a step more, and by
    any amount (infinity, and what comes of it) where h and d reach past the type."""
    return torch.where(h.abs() + d >= MOST[dtype], math.inf, d + HALF[dtype] * (h.abs() + d) + TINY[dtype])


# ---------------------------------------------------------------- routing


def route_ref(logits, k, normalize):
    """One token after the other: ids, weights (float64), offsets, rows, places."""
    x = logits.double().numpy()
    tokens, experts = x.shape
    ids, w = np.full((tokens, k), -1, np.int32), np.zeros((tokens, k))
    for t in range(tokens):
        ok = [e for e in range(experts) if x[t, e] > -math.inf]  # neither -infinity nor NaN
        if not ok:
            continue
        top = max(x[t, e] for e in ok)
        p = {e: 1.0 if x[t, e] == top else math.exp(x[t, e] - top) for e in ok}
        best = sorted(ok, key=lambda e: (-x[t, e], e))[:k]
        total = sum(p[e] for e in (best if normalize else ok))
        for j, e in enumerate(best):
            ids[t, j], w[t, j] = e, p[e] / total
    flat = ids.reshape(-1)
    offsets, rows, places = [0], [], np.full(tokens * k, -1, np.int32)
    for e in range(experts):
        mine = np.nonzero(flat == e)[0]
        places[mine] = len(rows) + np.arange(len(mine))
        rows += mine.tolist()
        offsets.append(len(rows))
    rows += [-1] * (tokens * k - len(rows))
    return {"ids": ids, "weights": w, "offsets": np.array(offsets, np.int32), "rows": np.array(rows, np.int32),
            "places": places}


# ---------------------------------------------------------------- products


def held(offsets, rows):
    """Offsets held to 0 .. rows and to never decrease."""
    out, low = [], 0
    for o in offsets:
        low = max(low, min(max(int(o), 0), rows))
        out.append(low)
    return out


def counts_to_offsets(counts):
    return [0] + np.cumsum(counts).tolist()


def random_w4(experts, n, k, group, dtype, seed, zeros):
    """Codes of all kinds, scales of both signs and very different sizes, on the CPU."""
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 256, (experts, n, k // 2), generator=g, dtype=torch.uint8)
    scale = (torch.randn((experts, n, k // group), generator=g) * torch.exp(torch.randn((experts, n, k // group), generator=g))
             / math.sqrt(k)).to(DT[dtype])
    z = torch.randint(0, 16, (experts, n, k // group), generator=g, dtype=torch.uint8) if zeros else None
    return codes, scale, z


def w4_values(codes, scale, zeros):
    """(whole numbers, scales) of every weight, float64 [experts, n, k]."""
    e, n, half = codes.shape
    c = torch.empty((e, n, 2 * half), dtype=torch.float64)
    c[..., 0::2], c[..., 1::2] = (codes & 15).double(), (codes >> 4).double()
    group = 2 * half // scale.shape[2]
    z = torch.full(scale.shape, 8.0, dtype=torch.float64) if zeros is None else zeros.double()
    return c - z.repeat_interleave(group, 2), scale.double().repeat_interleave(group, 2)


def product_ref(x, w, offsets, y, rows=None, fan=1, bias=None, epi=0, spread=None):
    """(y, bound): float64 results, and how far results of y's type may be off. w float64 [E, N, K];
    spread [E, N, K]: what stands for |w| in the sums' rounding (default |w|).

    A sum of K products of which each partial sum is rounded to fp32 is off by at most
    (K + 4) U S, S = sum |x w| (bias, scale and the last addition in the 4). Gated:
    f(g, v) = silu(g) v with |silu'| <= 1.1, so 1.1 |v| dg + |silu(g)| dv (dg dv is counted
    by the larger of v and v + dv), and the exponential, sum, quotient and product by
    (|g| + 8) U each way; ReLU does not widen. Then the output's own rounding."""
    out, bound = y.double().clone(), torch.zeros(y.shape, dtype=torch.float64)
    ends = held(offsets, y.shape[0])
    for e in range(w.shape[0]):
        p0, p1 = ends[e], ends[e + 1]
        if p0 == p1:
            continue
        src = torch.arange(p0, p1)
        if rows is not None:
            r = torch.as_tensor(rows)[p0:p1].long()
            src = torch.where(r >= 0, torch.div(r, fan, rounding_mode="floor"), -1)
        xd = torch.zeros((p1 - p0, w.shape[2]), dtype=torch.float64)
        there = (src >= 0) & (src < x.shape[0])
        xd[there] = x[src[there]].double()
        we = w[e]
        h = xd @ we.T
        s = xd.abs() @ (we.abs() if spread is None else spread[e]).T
        if bias is not None:
            h = h + bias[e].double()
            s = s + bias[e].double().abs()
        d = (w.shape[2] + 4) * U * s
        if epi & RELU:
            h = h.clamp(min=0)
        if epi & GATE:
            n = h.shape[1] // 2
            g, v, dg, dv = h[:, :n], h[:, n:], d[:, :n], d[:, n:]
            f = g / (1.0 + torch.exp(-g))
            h = f * v
            d = 1.1 * (v.abs() + dv) * dg + f.abs() * dv + (g.abs() + 8) * U * h.abs()
        out[p0:p1] = h
        bound[p0:p1] = rounded(h, d, y.dtype)
    return out, bound


class Weights4:
    """Weights of 4-bit codes, an expert at a time, as product_ref takes them; spread: what stands for |w|
    in the sums' rounding where sum x (B + code) and sum x are taken apart, at B = 16 (bf16) and 128 (fp16)."""

    def __init__(self, codes, scale, zeros, spread=0):
        self.parts, self.spread = (codes, scale, zeros), spread
        self.shape = (codes.shape[0], codes.shape[1], 2 * codes.shape[2])

    def __getitem__(self, e):
        codes, scale, zeros = self.parts
        z = None if zeros is None else zeros[e:e + 1]
        whole, s = w4_values(codes[e:e + 1], scale[e:e + 1], z)
        if not self.spread:
            return (whole * s)[0]
        zero = 8.0 if z is None else z.double().repeat_interleave(self.shape[2] // scale.shape[2], 2)
        return ((self.spread + zero) * s.abs())[0]


# ---------------------------------------------------------------- which kernel runs a product


class GroupedArgs(ctypes.Structure):
    """pyc_grouped of csrc/kernels/grouped_args.h."""
    _fields_ = [("x", ctypes.c_void_p), ("x_stride", ctypes.c_int64), ("x_rows", ctypes.c_int), ("rows", ctypes.c_void_p),
                ("fan", ctypes.c_int), ("offsets", ctypes.c_void_p), ("E", ctypes.c_int), ("P", ctypes.c_int),
                ("w", ctypes.c_void_p), ("w_stride", ctypes.c_int64), ("N", ctypes.c_int), ("K", ctypes.c_int),
                ("scale", ctypes.c_void_p), ("zeros", ctypes.c_void_p), ("group", ctypes.c_int), ("bias", ctypes.c_void_p),
                ("y", ctypes.c_void_p), ("y_stride", ctypes.c_int64), ("epi", ctypes.c_int)]


def form(w4, experts, rows, n, k, epi=0, x_rows=None, x_stride=None, dense=False, at=0x10000):
    """(kernel, its argument) of a call on 16-byte boundaries (at: another address of x): 0 general, 1 ring,
    2 tiles, 3 stream, 4 4-bit tiles."""
    out = n // 2 if epi & GATE else n
    g = GroupedArgs(at, k if x_stride is None else x_stride, rows if x_rows is None else x_rows, None, 1,
                    None if dense else 0x10000, experts, rows, 0x10000, n * (k // 2 if w4 else k), n, k, None, None, 0, None,
                    0x10000, out, epi)
    arg = ctypes.c_int(-1)
    f = pyc_amd.lib().pyc_hip_grouped_form
    f.argtypes = [ctypes.c_int, ctypes.POINTER(GroupedArgs), ctypes.POINTER(ctypes.c_int)]
    return f(int(w4), ctypes.byref(g), ctypes.byref(arg)), arg.value


def check(got, ref, bound):
    """Every element within its bound; says by how much the worst one uses it."""
    g = got.double().cpu()
    over = (g - ref).abs() - bound
    assert torch.isfinite(g[torch.isfinite(bound)]).all()
    assert not bool((over > 0).any()), f"off by {float((g - ref).abs().max())}, past the bound by {float(over.max())}"


def combine_ref(y, weights, places, base):
    """(out, bound): k products and sums in fp32 (at most k + 1 roundings of a partial sum,
    each at most U times the sum of magnitudes), then the output's own rounding."""
    t, k = weights.shape
    o = torch.zeros((t, y.shape[1]), dtype=torch.float64) if base is None else base.double().clone()
    s = o.abs()
    for i in range(t):
        for j in range(k):
            p = int(places[i * k + j])
            if 0 <= p < y.shape[0]:
                a = float(weights[i, j]) * y[p].double()
                o[i] += a
                s[i] += a.abs()
    return o, (k + 1) * U * s + HALF[y.dtype] * (o.abs() + (k + 1) * U * s) + TINY[y.dtype]
