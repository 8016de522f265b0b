"""GPU: products grouped by expert (pyc_hip_grouped_gemm_dispatch) against
moe_util.product_ref in 64 bits, bounds derived there."""
import math

import pytest

import pyc_amd
from tests import moe_util
from tests.moe_util import DT, GATE, RELU

pytestmark = pytest.mark.gpu


def _inputs(torch, counts, n, k, dtype, seed=0, extra=0):
    g = torch.Generator().manual_seed(seed + n + k)
    p = sum(counts) + extra
    x = torch.randn((p, k), generator=g).to(DT[dtype])
    w = (torch.randn((len(counts), n, k), generator=g) / math.sqrt(k)).to(DT[dtype])
    return x, w, moe_util.counts_to_offsets(counts)


def _i32(torch, v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _check(torch, x, w, offsets, n_out, rows=None, fan=1, bias=None, epi=0, p=None):
    y = torch.full((x.shape[0] if p is None else p, n_out), 7.0, dtype=x.dtype)
    ref, bound = moe_util.product_ref(x, w.double(), offsets, y, rows, fan, bias, epi)
    d = y.cuda()
    pyc_amd.grouped_gemm(x.cuda(), w.cuda(), _i32(torch, offsets), d, rows=None if rows is None else _i32(torch, rows), fan=fan,
                         bias=None if bias is None else bias.cuda(), epilogue=epi)
    moe_util.check(d, ref, bound)
    ends = moe_util.held(offsets, y.shape[0])
    assert (d[:ends[0]] == 7).all() and (d[ends[-1]:] == 7).all()
    return d


COUNTS = [[1], [0, 1, 0], [3, 0, 5, 1], [16, 17, 15], [0, 0, 0], [33, 2, 70, 0, 1], [130, 1, 64, 65]]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("counts", COUNTS, ids=str)
@pytest.mark.parametrize("n,k", [(64, 64), (128, 256), (40, 72), (33, 131), (1, 1), (200, 8), (7, 1000)])
def test_sizes(gpu, counts, n, k, dtype):
    _check(gpu, *_inputs(gpu, counts, n, k, dtype), n)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("epi", [0, RELU, GATE])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("n,k", [(96, 128), (50, 40), (2, 33), (512, 64)])
def test_epilogues(gpu, n, k, epi, bias, dtype):
    x, w, o = _inputs(gpu, [5, 0, 40, 2], n, k, dtype, extra=3)
    b = gpu.randn((4, n), generator=gpu.Generator().manual_seed(1)) if bias else None
    _check(gpu, x, w, o, n // 2 if epi == GATE else n, bias=b, epi=epi)


@pytest.mark.parametrize("n,k", [(64, 128), (36, 100)])
def test_gather(gpu, n, k):
    """A token's row goes to several experts; indexes outside x read zeros, the same index may come twice."""
    g = gpu.Generator().manual_seed(4)
    t, fan = 21, 3
    x = gpu.randn((t, k), generator=g).bfloat16()
    w = (gpu.randn((4, n, k), generator=g) / math.sqrt(k)).bfloat16()
    rows = gpu.randperm(t * fan, generator=g).tolist()
    rows[3], rows[10], rows[40], rows[41], rows[50] = -1, t * fan, 1 << 30, rows[42], -7
    bias = gpu.randn((4, n), generator=g)
    _check(gpu, x, w, [0, 20, 20, 55, 63], n, rows=rows, fan=fan, bias=bias, p=63)
    _check(gpu, x, w, [0, 20, 20, 55, 63], n // 2, rows=rows, fan=fan, epi=GATE, p=63)
    _check(gpu, x, w, [0, 20, 20, 55, 63], n, rows=None, p=63)  # rows of y past x: zeros


@pytest.mark.parametrize("offsets", [[5, 9, 9, 20, 30], [-3, 4, 2, 8, 60], [0, 100, 100, 100, 100], [40, 40, 40, 40, 40],
                                     [10, 0, 0, 0, 0], [0, 7, 3, 9, 9], [-5, -5, -5, -5, -5], [0, 0, 0, 0, 1 << 30]], ids=str)
def test_offsets_of_any_kind(gpu, offsets):
    """Held to the rows and to never decrease; rows outside every expert stay."""
    x, w, _ = _inputs(gpu, [10, 10, 10, 10], 64, 64, "bf16")
    _check(gpu, x, w, offsets, 64)
    x, w, _ = _inputs(gpu, [10, 10, 10, 10], 30, 35, "f16")
    _check(gpu, x, w, offsets, 30)


def test_many_experts(gpu):
    """More experts than lanes, most of them empty; and every one with a row."""
    counts = [0] * 200
    for e, c in ((0, 2), (63, 1), (64, 5), (127, 3), (199, 66)):
        counts[e] = c
    _check(gpu, *_inputs(gpu, counts, 32, 64, "bf16"), 32)
    _check(gpu, *_inputs(gpu, [1] * 130, 16, 32, "f16"), 16)
    _check(gpu, *_inputs(gpu, [0] * 1023 + [3], 8, 16, "f16"), 8)


@pytest.mark.parametrize("off", [0, 1, 4, 8])
def test_strides_and_alignment(gpu, off):
    """x, y and the experts' weights as parts of wider arrays, on 16 bytes and off them; nothing around y is written."""
    x, w, o = _inputs(gpu, [3, 20, 9], 48, 64, "bf16")
    xs = gpu.full((32, 80), 3.0, dtype=x.dtype, device="cuda")
    xs[:, off:off + 64] = x.cuda()
    ws = gpu.full((3, 48 * 64 + 40), 3.0, dtype=x.dtype, device="cuda")
    wv = ws[:, off:off + 48 * 64].view(3, 48, 64) if off == 0 else ws.as_strided((3, 48, 64), (48 * 64 + 40, 64, 1), off)
    wv.copy_(w.cuda())
    ys = gpu.full((32, 60), 5.0, dtype=x.dtype, device="cuda")
    pyc_amd.grouped_gemm(xs[:, off:off + 64], wv, _i32(gpu, o), ys[:, off:off + 48])
    ref, bound = moe_util.product_ref(x, w.double(), o, gpu.zeros((32, 48), dtype=x.dtype))
    moe_util.check(ys[:, off:off + 48], ref, bound)
    assert (ys[:, :off] == 5).all() and (ys[:, off + 48:] == 5).all()


def test_values_behind_the_operands(gpu):
    """NaN and infinity in x rows that no expert has, in weights of experts without rows and in what
    lies behind the last row do not reach a result."""
    x, w, o = _inputs(gpu, [4, 0, 6], 40, 72, "bf16", extra=5)
    x[10:] = float("nan")
    w[1] = float("inf")
    y = gpu.full((15, 40), 7.0, dtype=x.dtype, device="cuda")
    pyc_amd.grouped_gemm(x.cuda(), w.cuda(), _i32(gpu, o), y)
    keep = w.clone()
    keep[1] = 0
    ref, bound = moe_util.product_ref(gpu.nan_to_num(x), keep.double(), o, gpu.full((15, 40), 7.0, dtype=x.dtype))
    moe_util.check(y, ref, bound)
