"""GPU: products with 4-bit weights (pyc_hip_w4a16_gemm_dispatch and its form by expert)
against moe_util.product_ref in 64 bits. What stands for |w| in the sums' rounding: a
kernel may sum x (B + code) and x apart and take sum x (B + code) - (B + zero) sum x, with B up
to 16 in bf16 and 128 in fp16. Every partial sum of the first is at most (B + 15) sum |x|,
the second at most (B + zero) sum |x|, so the roundings are those of (2 B + 15 + zero)
|scale| |x| (64 + zero >= that in bf16, 272 + zero in fp16); scaling the groups' sums adds two
roundings that the bound's K + 4 holds."""
import pytest

import pyc_amd
from tests import moe_util
from tests.moe_util import DT, GATE, RELU

pytestmark = pytest.mark.gpu


def _i32(torch, v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _cuda(t):
    return None if t is None else t.cuda()


def _check(torch, x, codes, scale, zeros, offsets, n_out, rows=None, fan=1, bias=None, epi=0, p=None, dense=False):
    whole, s = moe_util.w4_values(codes, scale, zeros)
    z = 8.0 if zeros is None else zeros.double().repeat_interleave(whole.shape[2] // scale.shape[2], 2)
    y = torch.full((x.shape[0] if p is None else p, n_out), 7.0, dtype=x.dtype)
    ref, bound = moe_util.product_ref(x, whole * s, offsets, y, rows, fan, bias, epi, spread=((64 if x.dtype == torch.bfloat16 else 272) + z) * s.abs())
    d = y.cuda()
    if dense:
        pyc_amd.w4a16_gemm(x.cuda(), codes[0].cuda(), scale[0].cuda(), d, zeros=_cuda(None if zeros is None else zeros[0]),
                           bias=_cuda(None if bias is None else bias[0]), epilogue=epi)
    else:
        pyc_amd.w4a16_grouped_gemm(x.cuda(), codes.cuda(), scale.cuda(), _i32(torch, offsets), d, zeros=_cuda(zeros),
                                   rows=None if rows is None else _i32(torch, rows), fan=fan, bias=_cuda(bias), epilogue=epi)
    moe_util.check(d, ref, bound)
    return d


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m,n,k", [(1, 64, 128), (1, 1, 256), (2, 33, 384), (16, 130, 640), (17, 48, 1152), (31, 16, 128),
                                   (65, 70, 256), (200, 96, 384), (3, 260, 2048)])
def test_dense(gpu, m, n, k, group, dtype, zeros):
    g = gpu.Generator().manual_seed(m + n + k)
    x = gpu.randn((m, k), generator=g).to(DT[dtype])
    _check(gpu, x, *moe_util.random_w4(1, n, k, group, dtype, 3, zeros), [0, m], n, dense=True)


@pytest.mark.parametrize("k", [32, 64, 96, 160, 224, 416])
def test_short_and_odd_depths(gpu, k):
    """Depths that are no multiple of 128, with every group that divides them."""
    for group in (32, 64, 128):
        if k % group == 0:
            x = gpu.randn((5, k), generator=gpu.Generator().manual_seed(k)).bfloat16()
            _check(gpu, x, *moe_util.random_w4(1, 40, k, group, "bf16", 3, True), [0, 5], 40, dense=True)


@pytest.mark.parametrize("epi", [0, RELU, GATE])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("m", [1, 9, 80])
def test_epilogues(gpu, m, epi, bias):
    x = gpu.randn((m, 256), generator=gpu.Generator().manual_seed(m)).bfloat16()
    b = gpu.randn((1, 100), generator=gpu.Generator().manual_seed(1)) if bias else None
    _check(gpu, x, *moe_util.random_w4(1, 100, 256, 64, "bf16", 3, False), [0, m], 50 if epi == GATE else 100, bias=b,
           epi=epi, dense=True)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("counts", [[1], [0, 2, 0, 1], [3, 17, 0, 16, 33], [70, 0, 129]], ids=str)
@pytest.mark.parametrize("group,k", [(32, 96), (64, 256), (128, 384)])
def test_by_expert(gpu, counts, group, k, dtype):
    g = gpu.Generator().manual_seed(k)
    x = gpu.randn((sum(counts) + 2, k), generator=g).to(DT[dtype])
    w = moe_util.random_w4(len(counts), 72, k, group, dtype, 5, True)
    d = _check(gpu, x, *w, moe_util.counts_to_offsets(counts), 72)
    assert (d[sum(counts):] == 7).all()
    _check(gpu, x, *w, moe_util.counts_to_offsets(counts), 36, epi=GATE)


def test_gather(gpu):
    g = gpu.Generator().manual_seed(4)
    t, fan = 21, 3
    x = gpu.randn((t, 128), generator=g).bfloat16()
    w = moe_util.random_w4(4, 64, 128, 64, "bf16", 5, False)
    rows = gpu.randperm(t * fan, generator=g).tolist()
    rows[3], rows[10], rows[40], rows[41], rows[50] = -1, t * fan, 1 << 30, rows[42], -7
    _check(gpu, x, *w, [0, 20, 20, 55, 63], 64, rows=rows, fan=fan, p=63)
    _check(gpu, x, *w, [5, 30, 20, 55, 100], 32, rows=rows, fan=fan, p=63, epi=GATE)


def test_zero_points_of_any_byte(gpu):
    codes, scale, _ = moe_util.random_w4(1, 24, 128, 32, "f16", 6, False)
    zeros = gpu.randint(0, 256, scale.shape, generator=gpu.Generator().manual_seed(1), dtype=gpu.uint8)
    x = gpu.randn((4, 128), generator=gpu.Generator().manual_seed(2)).half()
    _check(gpu, x, codes, scale, zeros, [0, 4], 24, dense=True)


def test_strides(gpu):
    """x and y as parts of wider rows, experts apart; nothing around y is written."""
    x = gpu.randn((30, 128), generator=gpu.Generator().manual_seed(2)).bfloat16()
    codes, scale, zeros = moe_util.random_w4(3, 50, 128, 32, "bf16", 7, True)
    offsets = [0, 9, 28, 30]
    xs = gpu.full((30, 160), 3.0, dtype=x.dtype, device="cuda")
    xs[:, 16:144] = x.cuda()
    cs = gpu.full((3, 50 * 64 + 48), 255, dtype=gpu.uint8, device="cuda")
    cv = cs.as_strided((3, 50, 64), (50 * 64 + 48, 64, 1), 16)
    cv.copy_(codes.cuda())
    for off in (0, 3, 8):
        ys = gpu.full((30, 60), 5.0, dtype=x.dtype, device="cuda")
        pyc_amd.w4a16_grouped_gemm(xs[:, 16:144], cv, scale.cuda(), _i32(gpu, offsets), ys[:, off:off + 50], zeros=zeros.cuda())
        whole, s = moe_util.w4_values(codes, scale, zeros)
        ref, bound = moe_util.product_ref(x, whole * s, offsets, gpu.zeros((30, 50), dtype=x.dtype), spread=80 * s.abs())
        moe_util.check(ys[:, off:off + 50], ref, bound)
        assert (ys[:, :off] == 5).all() and (ys[:, off + 50:] == 5).all()
