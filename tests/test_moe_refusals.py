"""CPU: what the entry points of expert layers and 4-bit weights refuse, before any
launch, and the 64-bit restatements that the GPU tests compare with, by hand."""
import math

import numpy as np
import pytest
import torch

import pyc_amd
from tests import moe_util

P = 0x10000  # a non-null pointer on a 16-byte boundary, never read


def _route(symbol=b"hip_moe_route_f32", tokens=100, experts=8, k=2, logits=P, stride=8, ids=P, weights=P, offsets=P, rows=P,
           places=P, ws=P, ws_bytes=1 << 30):
    return pyc_amd.lib().pyc_hip_moe_route_dispatch(symbol, tokens, experts, k, 1, logits, stride, ids, weights, offsets, rows,
                                                    places, ws, ws_bytes, None)


def _combine(symbol=b"hip_moe_combine_bf16", rows=8, tokens=4, k=2, width=64, y=P, ys=64, weights=P, places=P, base=P, bs=64,
             out=P, os=64):
    return pyc_amd.lib().pyc_hip_moe_combine_dispatch(symbol, rows, tokens, k, width, y, ys, weights, places, base, bs, out, os,
                                                      None)


def _grouped(symbol=b"hip_grouped_gemm_bf16", experts=4, rows=8, N=64, K=32, x=P, xs=32, x_rows=8, src=None, fan=1, offsets=P,
             w=P, ws=64 * 32, bias=None, epi=0, y=P, ys=64):
    return pyc_amd.lib().pyc_hip_grouped_gemm_dispatch(symbol, experts, rows, N, K, x, xs, x_rows, src, fan, offsets, w, ws,
                                                       bias, epi, y, ys, None)


def _w4(symbol=b"hip_gemm_w4a16_bf16", M=8, N=64, K=128, group=64, x=P, xs=128, codes=P, scale=P, zeros=None, bias=None,
        epi=0, y=P, ys=64):
    return pyc_amd.lib().pyc_hip_w4a16_gemm_dispatch(symbol, M, N, K, group, x, xs, codes, scale, zeros, bias, epi, y, ys, None)


def _w4_grouped(symbol=b"hip_grouped_gemm_w4a16_f16", experts=4, rows=8, N=64, K=128, group=64, x=P, xs=128, x_rows=8,
                src=None, fan=1, offsets=P, codes=P, cs=64 * 64, scale=P, zeros=None, bias=None, epi=0, y=P, ys=64):
    return pyc_amd.lib().pyc_hip_w4a16_grouped_gemm_dispatch(symbol, experts, rows, N, K, group, x, xs, x_rows, src, fan,
                                                             offsets, codes, cs, scale, zeros, bias, epi, y, ys, None)


@pytest.mark.parametrize("bad", [dict(symbol=b"hip_moe_route"), dict(symbol=b"hip_moe_combine_bf16"), dict(symbol=None),
                                 dict(tokens=-1), dict(tokens=(1 << 22) + 1), dict(experts=0), dict(experts=1025, stride=2000),
                                 dict(k=0), dict(k=9), dict(k=65, experts=100, stride=100), dict(logits=None),
                                 dict(logits=P + 2), dict(symbol=b"hip_moe_route_bf16", logits=P + 1), dict(stride=7),
                                 dict(ids=None), dict(weights=None), dict(offsets=None), dict(rows=None), dict(places=None),
                                 dict(ids=P + 2), dict(offsets=P + 1), dict(ws=None), dict(ws=P + 2), dict(ws_bytes=64),
                                 dict(tokens=0, offsets=None)], ids=str)
def test_route_refusals(bad):
    assert _route(**bad) == -1


@pytest.mark.parametrize("bad", [dict(symbol=b"hip_moe_combine_f32"), dict(symbol=None), dict(rows=-1),
                                 dict(rows=(1 << 28) + 1), dict(tokens=-1), dict(tokens=(1 << 22) + 1), dict(k=0), dict(k=65),
                                 dict(width=0), dict(width=(1 << 24) + 1), dict(y=None), dict(y=P + 1), dict(ys=63),
                                 dict(weights=None), dict(weights=P + 2), dict(places=None), dict(base=P + 1), dict(bs=60),
                                 dict(out=None), dict(out=P + 1), dict(os=10),
                                 dict(tokens=1 << 16, width=1 << 16, ys=1 << 16, bs=1 << 16, os=1 << 16),
                                 dict(tokens=1 << 22, width=1 << 16, ys=1 << 16, bs=1 << 16, os=1 << 16)], ids=str)
def test_combine_refusals(bad):
    assert _combine(**bad) == -1


PRODUCT = [dict(symbol=None), dict(symbol=b"hip_gemm_bf16_nt"), dict(N=0), dict(K=0), dict(N=(1 << 24) + 1), dict(x=None),
           dict(x=P + 1), dict(xs=16), dict(y=None), dict(y=P + 1), dict(ys=63), dict(epi=8), dict(epi=6),
           dict(epi=1), dict(epi=1, bias=P + 2), dict(epi=4, N=63), dict(epi=-1)]
BY_EXPERT = [dict(experts=0), dict(experts=1025), dict(rows=-1), dict(rows=(1 << 28) + 1), dict(x_rows=-1),
             dict(x_rows=(1 << 28) + 1), dict(fan=0), dict(src=P + 2), dict(offsets=None), dict(offsets=P + 1)]
FOUR_BITS = [dict(group=16), dict(group=0), dict(group=96), dict(K=160, xs=160), dict(codes=None), dict(codes=P + 8),
             dict(scale=None), dict(scale=P + 1), dict(x=P + 8), dict(xs=129)]


@pytest.mark.parametrize("bad", PRODUCT + BY_EXPERT + [dict(w=None), dict(w=P + 1), dict(ws=64 * 32 - 1)], ids=str)
def test_grouped_refusals(bad):
    assert _grouped(**bad) == -1


@pytest.mark.parametrize("bad", PRODUCT + FOUR_BITS + [dict(M=-1), dict(M=(1 << 28) + 1)], ids=str)
def test_w4_refusals(bad):
    assert _w4(**bad) == -1


@pytest.mark.parametrize("bad", PRODUCT + BY_EXPERT + FOUR_BITS + [dict(cs=64 * 64 - 16), dict(cs=64 * 64 + 8)], ids=str)
def test_w4_grouped_refusals(bad):
    assert _w4_grouped(**bad) == -1


def test_nothing_to_do():
    """No rows, no tokens: nothing is launched, operands may be null."""
    assert _combine(tokens=0, y=None, weights=None, places=None, base=None, out=None) == 0
    assert _grouped(rows=0, x=None, w=None, y=None, offsets=None) == 0
    assert _w4(M=0, x=None, codes=None, scale=None, y=None) == 0
    assert _w4_grouped(rows=0, x=None, codes=None, scale=None, y=None, offsets=None) == 0


def test_workspace_sizes():
    f = pyc_amd.lib().pyc_hip_moe_route_workspace
    for e, k in ((1, 1), (8, 2), (128, 8), (1024, 64)):
        sizes = [f(t, e, k) for t in list(range(0, 200)) + [1000, 8192, 1 << 22]]
        assert all(0 < a <= b for a, b in zip(sizes, sizes[1:]))
    for bad in ((-1, 8, 2), ((1 << 22) + 1, 8, 2), (8, 0, 1), (8, 1025, 1), (8, 8, 0), (8, 8, 9), (8, 100, 65)):
        assert f(*bad) == 0, bad


def test_wrapper_refusals():
    """The Python wrappers refuse host tensors and tensors of other types and shapes before they reach the library."""
    i32 = lambda *n: torch.zeros(n, dtype=torch.int32)  # noqa: E731
    h = lambda *n: torch.zeros(n, dtype=torch.bfloat16)  # noqa: E731
    u8 = lambda *n: torch.zeros(n, dtype=torch.uint8)  # noqa: E731
    for call in (lambda: pyc_amd.moe_route(torch.zeros((4, 8)), i32(4, 2), torch.zeros((4, 2)), i32(9), i32(8), i32(8)),
                 lambda: pyc_amd.moe_combine(h(8, 16), torch.zeros((4, 2)), i32(8), h(4, 16)),
                 lambda: pyc_amd.grouped_gemm(h(8, 16), h(2, 4, 16), i32(3), h(8, 4)),
                 lambda: pyc_amd.grouped_gemm(h(8, 16), h(4, 16), i32(3), h(8, 4)),
                 lambda: pyc_amd.w4a16_gemm(h(8, 64), u8(4, 32), h(4, 1), h(8, 4)),
                 lambda: pyc_amd.w4a16_gemm(h(8, 64), u8(4, 32), h(1, 4, 1), h(8, 4)),
                 lambda: pyc_amd.w4a16_grouped_gemm(h(8, 64), u8(2, 4, 32), h(2, 4, 1), i32(3), h(8, 4)),
                 lambda: pyc_amd.w4a16_grouped_gemm(h(8, 64), u8(4, 32), h(2, 4, 1), i32(3), h(8, 4))):
        with pytest.raises(pyc_amd.PycError):
            call()


def test_registered():
    L = pyc_amd.lib()
    for key, n in (("moe_route", 3), ("moe_combine", 2), ("grouped_gemm", 2), ("matmul_w4a16", 2), ("grouped_w4a16", 2)):
        assert L.pyc_hip_kernel_symbol_count(key.encode()) == n
    for sym in ("hip_moe_route_f32", "hip_moe_route_bf16", "hip_moe_route_f16", "hip_moe_combine_bf16", "hip_moe_combine_f16",
                "hip_grouped_gemm_bf16", "hip_grouped_gemm_f16", "hip_gemm_w4a16_bf16", "hip_gemm_w4a16_f16",
                "hip_grouped_gemm_w4a16_bf16", "hip_grouped_gemm_w4a16_f16"):
        assert pyc_amd.kernel_resources(sym).threads > 0


def test_route_restatement_by_hand():
    """Three tokens: a tie, a padded one, one with a single expert left."""
    inf = math.inf
    x = torch.tensor([[0.0, 1.0, 1.0], [-inf, -inf, -inf], [-inf, -inf, 5.0]])
    r = moe_util.route_ref(x, 2, True)
    assert r["ids"].tolist() == [[1, 2], [-1, -1], [2, -1]]
    assert r["weights"].tolist() == [[0.5, 0.5], [0, 0], [1, 0]]
    assert r["offsets"].tolist() == [0, 0, 1, 3] and r["rows"].tolist() == [0, 1, 4, -1, -1, -1]
    assert r["places"].tolist() == [0, 1, -1, -1, 2, -1]
    full = moe_util.route_ref(x, 2, False)["weights"][0]
    assert abs(full[0] - math.e / (2 * math.e + 1)) < 1e-15


def test_product_restatement_by_hand():
    x = torch.tensor([[1.0, 2.0], [3.0, -1.0]]).bfloat16()
    w = torch.tensor([[[1.0, 1.0], [0.0, 1.0]], [[2.0, 0.0], [1.0, -1.0]]], dtype=torch.float64)
    y, _ = moe_util.product_ref(x, w, [0, 1, 2], torch.zeros((3, 2), dtype=torch.bfloat16))
    assert y.tolist() == [[3.0, 2.0], [6.0, 4.0], [0.0, 0.0]]
    g, _ = moe_util.product_ref(x, w, [0, 1, 2], torch.zeros((2, 1), dtype=torch.bfloat16), epi=moe_util.GATE)
    assert abs(float(g[1, 0]) - 6.0 / (1 + math.exp(-6.0)) * 4.0) < 1e-12
    assert moe_util.held([3, 1, 9, -2, 50], 10) == [3, 3, 9, 9, 10]


def test_w4_restatement_by_hand():
    codes = torch.tensor([[[0x80, 0xF1]]], dtype=torch.uint8)
    whole, s = moe_util.w4_values(codes, torch.tensor([[[0.5, 2.0]]]), torch.tensor([[[1, 3]]], dtype=torch.uint8))
    assert (whole * s).tolist() == [[[-0.5, 3.5, -4.0, 24.0]]]
    whole, _ = moe_util.w4_values(codes, torch.tensor([[[0.5, 2.0]]]), None)
    assert np.array_equal(whole[0, 0].numpy(), [-8, 0, -7, 7])
