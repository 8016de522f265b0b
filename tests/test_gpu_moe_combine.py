"""GPU: the weighted sum of experts' rows (pyc_hip_moe_combine_dispatch) against
moe_util.combine_ref in 64 bits."""
import pytest

import pyc_amd
from tests import moe_util
from tests.moe_util import DT

pytestmark = pytest.mark.gpu


def _inputs(torch, t, k, h, dtype, base, seed=0):
    g = torch.Generator().manual_seed(seed + t * 100 + h)
    y = torch.randn((t * k, h), generator=g).to(DT[dtype])
    w = torch.rand((t, k), generator=g)
    places = torch.randperm(t * k, generator=g).to(torch.int32)
    b = torch.randn((t, h), generator=g).to(DT[dtype]) if base else None
    return y, w, places, b


@pytest.mark.parametrize("base", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("t,k,h", [(1, 1, 1), (1, 8, 64), (3, 2, 2048), (32, 8, 1000), (7, 9, 129), (5, 17, 24), (2, 64, 8),
                                   (333, 4, 56)])
def test_sizes(gpu, t, k, h, dtype, base):
    y, w, p, b = _inputs(gpu, t, k, h, dtype, base)
    out = gpu.full((t, h), 9.0, dtype=y.dtype, device="cuda")
    pyc_amd.moe_combine(y.cuda(), w.cuda(), p.cuda(), out, base=None if b is None else b.cuda())
    moe_util.check(out, *moe_util.combine_ref(y, w, p, b))


@pytest.mark.parametrize("h", [40, 37])
def test_places_outside(gpu, h):
    """Absent choices are not read, whatever their weight: NaN and infinity weights on them,
    NaN in the rows nobody has."""
    y, w, p, b = _inputs(gpu, 9, 3, h, "bf16", True)
    y[int(p[4])] = float("nan")
    p[4], p[5], p[7] = -1, 27, 1 << 30
    w[1, 1] = float("nan")
    w[1, 2] = float("inf")
    p[18:21] = -1
    out = gpu.empty((9, h), dtype=y.dtype, device="cuda")
    pyc_amd.moe_combine(y.cuda(), w.cuda(), p.cuda(), out, base=b.cuda())
    ref, bound = moe_util.combine_ref(y, w, p, b)
    assert gpu.isfinite(out).all()
    moe_util.check(out, ref, bound)
    assert gpu.equal(out[6].cpu(), b[6])
    none = gpu.empty((9, h), dtype=y.dtype, device="cuda")
    pyc_amd.moe_combine(y.cuda()[:0], w.cuda(), p.cuda(), none)
    assert (none == 0).all()


def test_strides_and_place(gpu):
    """Rows inside wider ones at odd and even places; out may be base; nothing around it is written."""
    for h, off in ((64, 8), (64, 3), (33, 8)):
        y, w, p, b = _inputs(gpu, 20, 2, h, "f16", True)
        ys = gpu.zeros((40, 100), dtype=y.dtype, device="cuda")
        ys[:, off:off + h] = y.cuda()
        outs = gpu.full((20, 120), 5.0, dtype=y.dtype, device="cuda")
        outs[:, off:off + h] = b.cuda()
        pyc_amd.moe_combine(ys[:, off:off + h], w.cuda(), p.cuda(), outs[:, off:off + h], base=outs[:, off:off + h])
        moe_util.check(outs[:, off:off + h], *moe_util.combine_ref(y, w, p, b))
        assert (outs[:, :off] == 5).all() and (outs[:, off + h:] == 5).all()


def test_no_tokens(gpu):
    e = gpu.empty((0, 8), dtype=gpu.bfloat16, device="cuda")
    pyc_amd.moe_combine(e, gpu.empty((0, 2), device="cuda"), gpu.empty(0, dtype=gpu.int32, device="cuda"), e)
