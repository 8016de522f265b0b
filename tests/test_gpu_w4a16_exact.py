"""4-bit products whose sums are exact (moe_exact), in every kernel and at every depth of the list of forms: results are
equal to the formula's. A wrong scale, zero point or group cannot hide in the rounding of a deep sum; CPU tests
plant each of these mistakes in the formula and see it found."""
import pytest
import torch

from tests import moe_exact, moe_util
from tests.moe_util import GATE, RELU
from tests.test_gpu_grouped_forms import FOUR


def _kinds(counts, n, k):
    """The plain call; gated, through an index with repeats and places outside x, with a bias; ReLU."""
    p = sum(counts)
    bias = moe_exact.biases(len(counts), n, n + k)
    rows = torch.randint(-2, 2 * p, (p,), generator=torch.Generator().manual_seed(k)).tolist()
    rows[0], rows[-1] = 1 << 30, 2 * p - 1
    return [dict(), dict(epi=GATE, rows=rows, fan=2, bias=bias), dict(epi=RELU, bias=bias), dict(epi=GATE)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("kind,arg,counts,n,depths", FOUR)
def test_every_form(gpu, kind, arg, counts, n, depths, group, dtype):
    for k in depths[group]:
        x, offsets = moe_exact.rows_of_x(sum(counts), k, dtype, n), moe_util.counts_to_offsets(counts)
        for zeros in (False, True):
            w = moe_exact.weights(len(counts), n, k, group, dtype, n + k, zeros)
            for kw in _kinds(counts, n, k):
                moe_exact.run(x, w, offsets, sum(counts), n, **kw)
                if len(counts) == 1 and "rows" not in kw:
                    moe_exact.run(x, w, offsets, sum(counts), n, dense=True, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows", [1, 5, 16, 23])
def test_streamed_turns(gpu, rows, group, dtype):
    """One row to some through deep products of few and many columns: x and scales through LDS in one turn and in several, with
    turns that end inside the row, and x beside the weights."""
    for n, k in ((40, 11008), (528, 7168), (4104, 2176), (33, 1920)):
        x, w = moe_exact.rows_of_x(rows, k, dtype, k), moe_exact.weights(1, n, k, group, dtype, n, True)
        assert moe_util.form(True, 1, rows, n, k, dense=True)[0] == 3
        moe_exact.run(x, w, [0, rows], rows, n, dense=True)


# ---------------------------------------------------------------- mistakes that the comparison has to find


def _mistakes(codes, scale, zeros, x, group):
    """(name, weights, x) with one thing wrong, as a kernel's slip at the edge of a group or turn would have it."""
    groups = scale.shape[2]
    for q in sorted({0, groups // 2, groups - 1}):
        no = x.clone()
        no[:, q * group:(q + 1) * group] = 0
        yield f"group {q} left out", (codes, scale, zeros), no
        if groups > 1:
            other = scale.clone()
            other[:, :, q] = scale[:, :, q - 1]
            yield f"scale of group {q} from the one before", (codes, other, zeros), x
        z = zeros.clone()
        z[:, :, q] += 1
        yield f"zero point of group {q} one more", (codes, scale, z), x
    no = x.clone()
    no[:, (x.shape[1] - 1) // 128 * 128:] = 0
    yield "last chunk of 128 left out", (codes, scale, zeros), no
    yield "halves of a byte changed", (codes >> 4 | codes << 4, scale, zeros), x
    yield "no zero points", (codes, scale, None), x
    yield "scales of the row before", (codes, scale.roll(1, 1), zeros), x
    yield "all zeros", (codes, scale, zeros), torch.zeros_like(x)


@pytest.mark.parametrize("epi", [0, GATE])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("rows,k,group", [(3, 7200, 32), (32, 11008, 32), (32, 4160, 64), (32, 3584, 128), (10, 6016, 128),
                                          (70, 448, 64), (70, 96, 32), (70, 128, 128)])
def test_mistakes_are_found(rows, k, group, dtype, epi):
    n = 8
    w, x = moe_exact.weights(1, n, k, group, dtype, k, True), moe_exact.rows_of_x(rows, k, dtype, rows)
    y = torch.full((rows, n // 2 if epi else n), 7.0, dtype=x.dtype)
    ref, bound = moe_exact.product(x, w, [0, rows], y, epi=epi)
    assert not moe_exact.wrong(ref.to(y.dtype), ref, bound).any()
    for name, wrong_w, wrong_x in _mistakes(*w, x, group):
        got, _ = moe_exact.product(wrong_x, wrong_w, [0, rows], y, epi=epi)
        bad = moe_exact.wrong(got.to(y.dtype), ref, bound).double().mean()
        assert bad > 0.1, (name, float(bad))


def test_sums_are_exact():
    """The largest sums there can be, taken in fp32 in another order and in two parts, are the formula's."""
    k, group = moe_exact.MOST_K, 32
    x = torch.full((1, k), 2.0)
    codes, scale = torch.full((1, 1, k // 2), 255, dtype=torch.uint8), torch.full((1, 1, k // group), 2.0 ** -5)
    whole, s = moe_util.w4_values(codes, scale, torch.zeros_like(scale))
    parts = (x * (16 + whole[0]).float()).view(-1, group).sum(1) * scale[0, 0], x.view(-1, group).sum(1) * 16 * scale[0, 0]
    a, b = (torch.cumsum(p.flip(0), 0)[-1] for p in parts)
    assert float(a - b) == float((x.double() * whole[0] * s[0]).sum())
    assert float(a) / moe_exact.STEP < 2 ** 24
