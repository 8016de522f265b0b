"""GPU: routing of many tokens, where the second launch's workgroups add up thousands of blocks' words, against whole
tensor operations in 64 bits (a stable sort: ties to the lower expert)."""
import pytest
import torch

import pyc_amd
from tests.moe_util import DT, U

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t,e,k,dtype", [(100_003, 128, 8, "bf16"), (70_000, 300, 3, "f32"), (262_145, 16, 2, "f16")])
def test_many_tokens(gpu, t, e, k, dtype):
    g = torch.Generator().manual_seed(t)
    x = (torch.randn((t, e), generator=g) * 2).to(DT[dtype])
    x[-5:] = -torch.inf
    x[::7, :e // 2] = -torch.inf
    i32 = dict(dtype=torch.int32, device="cuda")
    ids, w = torch.full((t, k), 77, **i32), torch.full((t, k), 7.0, device="cuda")
    offsets, rows, places = torch.full((e + 1,), 77, **i32), torch.full((t * k,), 77, **i32), torch.full((t * k,), 77, **i32)
    pyc_amd.moe_route(x.cuda(), ids, w, offsets, rows, places, normalize=False)

    v, order = torch.sort(x.double(), dim=1, descending=True, stable=True)
    there = v[:, :k] > -torch.inf
    want = torch.where(there, order[:, :k], -1)
    assert torch.equal(ids.cpu().long(), want)
    d = v - v[:, :1]  # of rows without a logit: NaN, not looked at
    p = torch.exp(d)[:, :k] / torch.exp(d).sum(1, keepdim=True)
    off = (w.cpu().double() - p).abs() - (2 * d[:, :k].abs() + 16) * U * p - 2.0 ** -126
    assert not bool((off > 0)[there].any()) and bool((w.cpu()[~there] == 0).all())

    flat = torch.where(there, order[:, :k], e).reshape(-1)
    by = torch.sort(flat, stable=True)[1]
    ends = torch.cumsum(torch.bincount(flat, minlength=e + 1), 0)
    assert offsets.tolist() == [0] + ends[:e].tolist()
    n = int(ends[e - 1])
    assert torch.equal(rows[:n].cpu().long(), by[:n]) and bool((rows[n:] == -1).all())
    at = torch.full((t * k,), -1)
    at[by[:n]] = torch.arange(n)
    assert torch.equal(places.cpu().long(), at)
