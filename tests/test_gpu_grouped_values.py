"""GPU: values at the ends of what the products by expert take, in every kernel of theirs: NaN and
infinity through ReLU, gates where e^-g comes near the end of fp32."""
import math

import pytest
import torch

import pyc_amd
from tests import moe_util
from tests.moe_util import DT, GATE, RELU, U

# (kernel, argument, rows of each expert, N, K) and, 4-bit, the group
SIXTEEN = [(0, 0, [30, 0, 64, 3], 1008, 63), (1, 1, [30, 0, 64, 3], 1008, 64), (1, 2, [300, 20, 270], 4112, 64),
           (2, 0, [700, 324], 8192, 64)]
FOUR = [(3, 0, [1, 0, 7, 2], 1040, 96, 32), (3, 0, [10], 96, 11008, 64), (4, 1, [90, 0, 107, 3], 1040, 128, 128),
        (4, 2, [200], 2000, 64, 32), (4, 4, [90, 0, 107, 3], 3600, 64, 64), (4, 0, [700], 8192, 128, 128)]
ALL = [(16, *c, 0) for c in SIXTEEN] + [(4, *c) for c in FOUR]


@pytest.mark.parametrize("bits,kind,arg,counts,n,k,group", ALL)
def test_which_kernel(bits, kind, arg, counts, n, k, group):
    for epi in (RELU, GATE):
        assert moe_util.form(bits == 4, len(counts), sum(counts), n, k, epi) == (kind, arg)


def _call(bits, x, w, counts, y, **kw):
    offsets = torch.tensor(moe_util.counts_to_offsets(counts), dtype=torch.int32, device="cuda")
    if bits == 16:
        pyc_amd.grouped_gemm(x, w, offsets, y, **kw)
    else:
        pyc_amd.w4a16_grouped_gemm(x, w[0], w[1], offsets, y, **kw)


def _weights(bits, e, n, k, group, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    if bits == 16:
        return (torch.randn((e, n, k), generator=g) / math.sqrt(k)).to(DT[dtype]).cuda()
    return [v.cuda() for v in moe_util.random_w4(e, n, k, group, dtype, seed, False)[:2]]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("bits,kind,arg,counts,n,k,group", ALL)
def test_relu_keeps_nan(gpu, bits, kind, arg, counts, n, k, group, dtype):
    """max(v, 0) of NaN is NaN, from the sums as from the bias; of +infinity itself, of -infinity 0. Other results keep their bits."""
    g = torch.Generator().manual_seed(n)
    x = torch.randn((sum(counts), k), generator=g).to(DT[dtype]).cuda()
    w = _weights(bits, len(counts), n, k, group, dtype, 5)
    bias = torch.randn((len(counts), n), generator=g).cuda()
    y = [torch.full((sum(counts), n), 7.0, dtype=x.dtype, device="cuda") for _ in range(2)]
    _call(bits, x, w, counts, y[0], bias=bias, epilogue=RELU)
    assert torch.isfinite(y[0]).all() and (y[0] >= 0).all() and (y[0] == 0).any()
    bad = bias.clone()
    bad[:, 0::8], bad[:, 3::8], bad[:, 6::8] = math.nan, math.inf, -math.inf
    if bits == 16:
        w = w.clone()
        w[:, 5::8, 0] = math.nan
    else:
        w[1][:, 5::8, 0] = math.nan
    _call(bits, x, w, counts, y[1], bias=bad, epilogue=RELU)
    assert torch.isnan(y[1][:, 0::8]).all() and torch.isnan(y[1][:, 5::8]).all()
    assert (y[1][:, 3::8] == math.inf).all() and (y[1][:, 6::8] == 0).all()
    for c in (1, 2, 4, 7):
        assert torch.equal(y[0][:, c::8], y[1][:, c::8])


def _gates(n):
    """n gates: all over -100 .. 100, more of them where 1 + e^-g is past 2^126, and odd ones."""
    odd = [0.0, -0.0, 1e-30, -1e-30, 2.0 ** -126, -(2.0 ** -126), 1e4, -1e4, 3e37, -3e37]
    a = torch.linspace(-100, 100, (n - len(odd)) // 2, dtype=torch.float64)
    b = torch.linspace(-88.9, -87.0, n - len(odd) - a.numel(), dtype=torch.float64)
    return torch.cat([a, b, torch.tensor(odd, dtype=torch.float64)]).float()


def _gate_ref(g, v, dtype):
    """silu(g) v, and how far it may be off: (|g| + 8) U of itself and the output's rounding. Where e^-g
    leaves fp32, below -88.722, silu(g) counts as 0."""
    g, v = g.double(), v.double()
    f = g / (1.0 + torch.exp(-g)) * v
    d = (g.abs() + 8) * U * f.abs()
    return f, moe_util.rounded(f, torch.where(g < -88.722, f.abs(), d), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("bits,kind,arg,counts,n,k,group", ALL)
def test_gates_near_the_end_of_fp32(gpu, bits, kind, arg, counts, n, k, group, dtype):
    """Gates and values by the bias alone (weights of zero). Large values, so that silu of -88 shows."""
    e, f = len(counts), n // 2
    gates = _gates(f)
    x = torch.randint(-2, 3, (sum(counts), k), generator=torch.Generator().manual_seed(n)).to(DT[dtype]).cuda()
    w = torch.zeros((e, n, k), dtype=DT[dtype], device="cuda") if bits == 16 else [
        torch.full((e, n, k // 2), 0x88, dtype=torch.uint8, device="cuda"), torch.ones((e, n, k // group), dtype=DT[dtype], device="cuda")]
    for value in (1.0, -3.0, 1e36):
        values = torch.where(gates > 80, 1.0, value)  # large ones for small results only
        bias = torch.cat([gates, values]).expand(e, n).contiguous().cuda()
        y = torch.full((sum(counts), f), 7.0, dtype=x.dtype, device="cuda")
        _call(bits, x, w, counts, y, bias=bias, epilogue=GATE)
        ref, bound = _gate_ref(gates, values, x.dtype)
        moe_util.check(y, ref.expand(sum(counts), f), bound.expand(sum(counts), f))


def test_gate_restatement_by_hand():
    g, v = torch.tensor([-88.0, -87.4, 0.0, 2.0]), torch.full((4,), 1e36)
    f, d = _gate_ref(g, v, torch.bfloat16)
    assert abs(float(f[0]) - -88.0 * math.exp(-88.0) * float(v[0])) < 1e-12
    assert float(d[0]) < abs(float(f[0])) * 2.0 ** -7 and float(d[1]) < abs(float(f[1])) * 2.0 ** -7  # 0 would not pass
