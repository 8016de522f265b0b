"""GPU: calls of experts' operators so large that one launch cannot hold their threads (2^32 - 1), with
whole numbers as operands, so that results are equal."""
import pytest
import torch

import pyc_amd
from tests import moe_util
from tests import moe_util

MOST = (1 << 32) - 1  # threads of a launch


def _ints(shape, low, high, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(low, high, shape, generator=g, device="cuda", dtype=torch.int8).to(dtype)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _same(y, part):
    """y [rows, n] equals part(rows a .. b) for all pieces of rows."""
    for a in range(0, y.shape[0], 64):
        assert torch.equal(y[a:a + 64], part(a, min(a + 64, y.shape[0])).to(y.dtype)), a


@pytest.mark.gpu
def test_sum_of_most_threads(gpu):
    """The weighted sum of odd rows at the largest tokens * width there may be: a thread for each column, in whole workgroups
    more than a launch has."""
    tokens, width = (1 << 16) + 1, (1 << 16) - 1
    assert tokens * width == MOST and (tokens * width + 255) // 256 * 256 > MOST
    y, w = _ints((5, width), -9, 10, torch.bfloat16, 1), _ints((tokens, 1), 1, 4, torch.float32, 2)
    g = torch.Generator(device="cuda").manual_seed(3)
    places = torch.randint(-1, 5, (tokens,), generator=g, device="cuda", dtype=torch.int32)
    base = _ints((tokens, width), -3, 4, torch.bfloat16, 4)
    want = lambda a, b: base[a:b].float() + w[a:b] * y[places[a:b].clamp(min=0).long()].float() * (places[a:b, None] >= 0)  # noqa: E731
    out = torch.full((tokens, width), 77.0, dtype=torch.bfloat16, device="cuda")
    pyc_amd.moe_combine(y, w, places, out, base=base)
    for a in range(0, tokens, 8192):
        assert torch.equal(out[a:a + 8192], want(a, a + 8192).bfloat16()), a
# (kernel, bits, N, K): 1024 experts of a row each
PRODUCTS = [(0, 16, 1 << 20, 1), (1, 16, 1 << 21, 8), (3, 4, 1 << 20, 32)]


@pytest.mark.parametrize("kind,bits,n,k", PRODUCTS)
def test_which_kernel(kind, bits, n, k):
    got, arg = moe_util.form(bits == 4, 1024, 1024, n, k)
    assert got == kind
    columns, rows, threads = {0: (64, 64, 256), 1: (64 * arg, 64, 256), 3: (4 * 32, 16, 512)}[kind]
    assert (1024 + 1024 // rows) * (n // columns) * threads > MOST


@pytest.mark.gpu
@pytest.mark.parametrize("kind,bits,n,k", PRODUCTS)
def test_products_of_most_workgroups(gpu, kind, bits, n, k):
    e, dtype = 1024, torch.float16
    x = _ints((e, k), -2, 3, dtype, 1)
    offsets = _i32(list(range(e + 1)))
    y = torch.full((e, n), 77.0, dtype=dtype, device="cuda")
    per = torch.arange(e, device="cuda") % 5 - 2  # what an expert adds to all of its weights
    if bits == 16:
        first = _ints((n, k), -2, 3, dtype, 2)
        w = torch.empty((e, n, k), dtype=dtype, device="cuda")
        for i in range(0, e, 64):
            w[i:i + 64] = first + per[i:i + 64, None, None].to(dtype)
        pyc_amd.grouped_gemm(x, w, offsets, y)
        values = first.float()
    else:
        codes = torch.randint(0, 256, (n, k // 2), generator=torch.Generator(device="cuda").manual_seed(2), device="cuda", dtype=torch.uint8)
        scale = torch.ones((e, n, k // 32), dtype=dtype, device="cuda")
        zeros = (8 - per).to(torch.uint8)[:, None, None].expand(e, n, k // 32).contiguous()
        pyc_amd.w4a16_grouped_gemm(x, codes.expand(e, n, k // 2).contiguous(), scale, offsets, y, zeros=zeros)
        values = torch.stack([codes & 15, codes >> 4], -1).reshape(n, k).float() - 8
    total = x.float().sum(1)
    _same(y, lambda a, b: x[a:b].float() @ values.t() + (per[a:b] * total[a:b])[:, None])
