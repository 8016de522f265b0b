"""4-bit products of which every sum is exact: x of -2 .. 2, scales of +-2^-8 .. 2^-5, zero points of 0 .. 15 and
biases in steps of 2^-8. A product x (16 + code) scale, and the same with the zero point, is a whole number of 2^-8 of at
most 2 * 31 * 2^3, and 11008 of them, or any part of them in any order, are below 2^24 of that step (5.5e6): fp32 holds
them. So whichever way a kernel sums, its result is the formula's, rounded to 16 bits once, and has to be equal to that;
only the gate's function may be off, by (|g| + 8) U."""
import torch

import pyc_amd
from tests import moe_util
from tests.moe_util import DT, GATE, RELU, U

STEP = 2.0 ** -8
MOST_K = 11008


def weights(experts, n, k, group, dtype, seed, zeros):
    """Codes of all kinds, scales and zero points (None: 8) on the CPU."""
    assert k <= MOST_K
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 256, (experts, n, k // 2), generator=g, dtype=torch.uint8)
    shape = (experts, n, k // group)
    sign = 2.0 * torch.randint(0, 2, shape, generator=g) - 1.0
    scale = (sign * STEP * 2.0 ** torch.randint(0, 4, shape, generator=g)).to(DT[dtype])
    return codes, scale, torch.randint(0, 16, shape, generator=g, dtype=torch.uint8) if zeros else None


def rows_of_x(rows, k, dtype, seed):
    return torch.randint(-2, 3, (rows, k), generator=torch.Generator().manual_seed(seed)).to(DT[dtype])


def biases(experts, n, seed):
    return torch.randint(-512, 513, (experts, n), generator=torch.Generator().manual_seed(seed)).float() * STEP


def product(x, w, offsets, y, rows=None, fan=1, bias=None, epi=0):
    """(y, bound): the formula in 64 bits over y's rows of experts, 0 where results have to be equal once rounded."""
    h, _ = moe_util.product_ref(x, moe_util.Weights4(*w), offsets, y if not epi & GATE else y.repeat(1, 2), rows, fan, bias, epi & RELU)
    bound = torch.zeros(y.shape, dtype=torch.float64)
    if epi & GATE:
        ends = moe_util.held(offsets, y.shape[0])
        g, v = h.chunk(2, 1)
        f = g / (1.0 + torch.exp(-g)) * v
        bound = moe_util.rounded(f, (g.abs() + 8) * U * f.abs(), y.dtype)
        h = f
        for part in (slice(0, ends[0]), slice(ends[-1], None)):
            h[part], bound[part] = y[part].double(), 0.0
    return h, bound


def wrong(got, ref, bound):
    """Elements that are not what they have to be."""
    got = got.cpu()
    off = (got.double() - ref).abs() > bound
    return torch.where(bound == 0, got != ref.to(got.dtype), off | got.isnan())


def check(got, ref, bound):
    bad = wrong(got, ref, bound)
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} wrong, the first at {bad.nonzero()[0].tolist()}"


def _cuda(t):
    return None if t is None else t.cuda()


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def run(x, w, offsets, p, n, dense=False, at=None, **kw):
    """A call against the formula; at: where x lies on the device."""
    rows, bias, epi = kw.get("rows"), kw.get("bias"), kw.get("epi", 0)
    y = torch.full((p, n // 2 if epi & GATE else n), 7.0, dtype=x.dtype)
    ref, bound = product(x, w, offsets, y, rows, kw.get("fan", 1), bias, epi)
    d, (c, s, z) = y.cuda(), [_cuda(v) for v in w]
    x = x.cuda() if at is None else at
    if dense:
        pyc_amd.w4a16_gemm(x, c[0], s[0], d, zeros=None if z is None else z[0], bias=None if bias is None else bias[0].cuda(),
                           epilogue=epi)
    else:
        pyc_amd.w4a16_grouped_gemm(x, c, s, _i32(offsets), d, zeros=z, rows=None if rows is None else _i32(rows),
                                   fan=kw.get("fan", 1), bias=_cuda(bias), epilogue=epi)
    check(d, ref, bound)
