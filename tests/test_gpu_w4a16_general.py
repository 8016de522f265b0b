"""4-bit products in the general kernel, which takes the calls that no descriptor holds: x of three rows over more
than 4 GiB. Every group, depths that end inside a step of 64, with and without zero points, every epilogue, both types;
sums are exact (moe_exact), so results are equal to the formula's."""
import pytest
import torch

from tests import moe_exact, moe_util
from tests.moe_util import DT, GATE, RELU

FAR = 1_100_000_000  # elements between rows of x
GENERAL = [30, 0, 40, 5]


@pytest.mark.parametrize("k", [32, 96, 128, 416])
def test_far_rows_need_the_general_kernel(k):
    assert moe_util.form(True, len(GENERAL), sum(GENERAL), 72, k, x_rows=3, x_stride=FAR)[0] == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_the_general_kernel(gpu, dtype):
    wide = torch.empty(2 * FAR + 416, dtype=DT[dtype], device="cuda")
    p, offsets = sum(GENERAL), moe_util.counts_to_offsets(GENERAL)
    for k in (32, 96, 128, 416):
        few = moe_exact.rows_of_x(3, k, dtype, k)
        at = wide.as_strided((3, k), (FAR, 1))
        at.copy_(few.cuda())
        rows = torch.randint(-1, 3 * 2 + 1, (p,), generator=torch.Generator().manual_seed(k)).tolist()
        for group in (32, 64, 128):
            if k % group:
                continue
            for zeros in (False, True):
                w = moe_exact.weights(len(GENERAL), 72, k, group, dtype, k, zeros)
                bias = moe_exact.biases(len(GENERAL), 72, k)
                for kw in (dict(), dict(epi=RELU, bias=bias), dict(epi=GATE), dict(epi=GATE, bias=bias)):
                    moe_exact.run(few, w, offsets, p, 72, at=at, rows=rows, fan=2, **kw)
