"""GPU: calls of experts' operators so large that one launch cannot hold their threads (2^32 - 1), with
whole numbers as operands, so that results are equal."""
import pytest
import torch

import pyc_amd
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
