"""GPU: routing (pyc_hip_moe_route_dispatch) against moe_util.route_ref in 64 bits.
Whole numbers are equal. A weight is a quotient of e^d, d = l - m exact to U |d|, by a
sum of at most 1024 such terms in fp32: off by at most (2 |d| + 16) U relative (an
exponential of 2 U, sums over lanes in 10 steps, a quotient), and a weight below
2^-126 by a step of the smallest."""
import math

import numpy as np
import pytest

import pyc_amd
from tests import moe_util
from tests.moe_util import DT, U

pytestmark = pytest.mark.gpu


def _out(torch, t, e, k):
    i = dict(dtype=torch.int32, device="cuda")
    return {"ids": torch.full((t, k), 77, **i), "weights": torch.full((t, k), 7.0, device="cuda"),
            "offsets": torch.full((e + 1,), 77, **i), "rows": torch.full((t * k,), 77, **i),
            "places": torch.full((t * k,), 77, **i)}


def _check(o, logits, k, normalize):
    ref = moe_util.route_ref(logits, k, normalize)
    for n in ("ids", "offsets", "rows", "places"):
        assert np.array_equal(o[n].cpu().numpy(), ref[n]), n
    x = logits.double().numpy()
    got, w = o["weights"].cpu().double().numpy(), ref["weights"]
    top = np.nanmax(np.where(np.isnan(x), -np.inf, x), 1, initial=-np.inf)
    for t in range(w.shape[0]):
        for j in range(k):
            e = ref["ids"][t, j]
            d = 0.0 if e < 0 or not math.isfinite(top[t]) or not math.isfinite(x[t, e]) else abs(x[t, e] - top[t])
            assert abs(got[t, j] - w[t, j]) <= (2 * d + 16) * U * w[t, j] + 2.0 ** -126, (t, j, got[t, j], w[t, j])


def _run(torch, logits, k, normalize, **kw):
    o = _out(torch, logits.shape[0], logits.shape[1], k)
    pyc_amd.moe_route(logits, *o.values(), normalize=normalize, **kw)
    torch.cuda.synchronize()
    return o


@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("t,e,k", [(1, 1, 1), (1, 8, 2), (3, 64, 8), (31, 65, 5), (32, 128, 8), (33, 100, 1), (64, 256, 8),
                                   (65, 257, 3), (96, 7, 7), (300, 1024, 10), (1, 1024, 64), (1000, 16, 4), (600, 2, 2)])
def test_sizes(gpu, dtype, t, e, k, normalize):
    """Tokens around the blocks of 32 and both forms; experts on both sides of what a lane
    holds; ties in 16 bits."""
    g = gpu.Generator().manual_seed(t * 1000 + e)
    x = (gpu.randn((t, e), generator=g) * 2).to(DT[dtype])
    _check(_run(gpu, x.cuda(), k, normalize), x, k, normalize)


@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("t", [40, 200])
def test_odd_values(gpu, t, normalize):
    """Equal rows, rows of -infinity, with one or two finite logits, NaN, +infinity, the types' ends."""
    e, k, inf = 24, 4, math.inf
    x = gpu.randn((t, e), generator=gpu.Generator().manual_seed(5))
    x[0] = 0.0
    x[1] = -inf
    x[2] = -inf
    x[2, 17] = 3.0
    x[3, :] = -inf
    x[3, 20], x[3, 4] = -1e30, -3e38
    x[4, 5] = math.nan
    x[5] = math.nan
    x[6, 7] = x[6, 3] = inf
    x[7] = inf
    x[8] = -3.4e38
    x[9, 0], x[9, 1] = 3.4e38, -3.4e38
    x[10] = math.nan
    x[10, 23] = -inf
    x[11, 12] = -0.0
    x[11, 13] = 0.0
    x[12, 3] = inf
    x[12, 4] = math.nan
    x[t - 3:] = -inf
    _check(_run(gpu, x.cuda(), k, normalize), x, k, normalize)


def test_all_masked(gpu):
    for t in (5, 333):
        x = gpu.full((t, 9), -math.inf)
        o = _run(gpu, x.cuda(), 3, True)
        _check(o, x, 3, True)
        assert (o["rows"] == -1).all() and (o["offsets"] == 0).all()


def test_strided_rows(gpu):
    """Logits as part of wider rows, at an odd place."""
    wide = gpu.randn((100, 50), generator=gpu.Generator().manual_seed(2)).bfloat16()
    x = wide[:, 3:40]
    _check(_run(gpu, wide.cuda()[:, 3:40], 6, True), x, 6, True)


def test_no_tokens(gpu):
    o = _out(gpu, 0, 12, 2)
    pyc_amd.moe_route(gpu.empty((0, 12), device="cuda"), *o.values())
    gpu.cuda.synchronize()
    assert (o["offsets"] == 0).all()


def test_many_tokens_of_one_expert(gpu):
    """Every token takes the same experts: the ranks run over all blocks."""
    x = gpu.zeros((2000, 40))
    x[:, 33] = 2.0
    x[:, 2] = 1.0
    _check(_run(gpu, x.cuda(), 2, True), x, 2, True)


def test_stream_workspace_and_repeats(gpu):
    """On another stream, with a kept workspace of any content made for more tokens: the same bits every time."""
    x = gpu.randn((700, 60), generator=gpu.Generator().manual_seed(3))
    ws = pyc_amd.moe_route_workspace(5000, 60, 4)
    ws.fill_(255)
    first = _run(gpu, x.cuda(), 4, True)
    _check(first, x, 4, True)
    side = gpu.cuda.Stream()
    xd = x.cuda()
    gpu.cuda.synchronize()
    for _ in range(3):
        with gpu.cuda.stream(side):
            o = _run(gpu, xd, 4, True, workspace=ws)
        for n in o:
            assert gpu.equal(o[n], first[n]), n
    o = _run(gpu, xd, 4, True, stream=side.cuda_stream)
    assert gpu.equal(o["rows"], first["rows"])


@pytest.mark.parametrize("t,e,k", [(2100, 1024, 20), (130, 100, 64), (2081, 1000, 1)])
def test_many_words(gpu, t, e, k):
    """So many words of bits that a workgroup of the second launch takes eight blocks; more choices than its threads."""
    x = (gpu.randn((t, e), generator=gpu.Generator().manual_seed(t)) * 2).bfloat16()
    _check(_run(gpu, x.cuda(), k, True), x, k, True)
