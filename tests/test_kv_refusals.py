"""CPU: what the paged cache's entry points refuse, before any launch, and the
64-bit restatements that the GPU tests compare with, on small cases by hand."""
import ctypes as C

import numpy as np
import pytest
import torch

import pyc_amd
from pyc_amd import abi
from tests import kv_util

P = 0x10000  # a non-null pointer on a 16-byte boundary, never read


def _cache(**kw):
    d = dict(k=P, v=P, k_scale=P, v_scale=P, k_block_stride=2 * 16 * 64, v_block_stride=2 * 16 * 64, num_blocks=4,
             kv_heads=2, block_size=16, head_dim=64)
    d.update(kw)
    return abi.KvCache(**d)


BAD_CACHES = [dict(k=None), dict(v=None), dict(k_scale=None), dict(v_scale=None), dict(k=P + 8), dict(v=P + 1),
              dict(k_scale=P + 2), dict(k_block_stride=2 * 16 * 64 - 16), dict(v_block_stride=2 * 16 * 64 + 8),
              dict(k_block_stride=1 << 31), dict(v_block_stride=1 << 40),
              dict(num_blocks=0), dict(num_blocks=-1), dict(num_blocks=1 << 28), dict(kv_heads=0), dict(block_size=8),
              dict(block_size=48), dict(block_size=256), dict(head_dim=96), dict(head_dim=256)]


def _append(cache, symbol=b"hip_kv_append_bf16", tokens=4, k=P, ks=128, v=P, vs=128, slots=P):
    return pyc_amd.lib().pyc_hip_kv_append_dispatch(symbol, C.byref(cache) if cache is not None else None, tokens, k, ks,
                                                    v, vs, slots, None)


def _attention(cache, symbol=b"hip_kv_attention_bf16", B=2, tokens=4, hq=4, max_q=2, max_len=0, q=P, qs=256, table=P,
               ts=8, width=8, lens=P, offsets=P, o=P, os=256, scale=0.125, ws=P, ws_bytes=1 << 40):
    return pyc_amd.lib().pyc_hip_kv_attention_dispatch(
        symbol, C.byref(cache) if cache is not None else None, B, tokens, hq, max_q, max_len, q, qs, table, ts, width,
        lens, offsets, o, os, scale, ws, ws_bytes, None)


def _plan(symbol=b"hip_kv_plan", B=2, width=8, ts=8, bs=16, tokens=4, cached=P, fresh=P, table=P, free=P, cap=4, count=P,
          lens=P, offsets=P, slots=P, positions=P, after=P):
    return pyc_amd.lib().pyc_hip_kv_plan_dispatch(symbol, B, width, ts, bs, tokens, cached, fresh, table, free, cap, count,
                                                  lens, offsets, slots, positions, after, None)


@pytest.mark.parametrize("bad", BAD_CACHES, ids=lambda b: "-".join(f"{k}={v}" for k, v in b.items()))
def test_bad_caches(bad):
    assert _append(_cache(**bad)) == -1
    assert _attention(_cache(**bad)) == -1


@pytest.mark.parametrize("bad", [dict(symbol=b"hip_kv_append_f32"), dict(symbol=b"hip_kv_plan"), dict(symbol=None),
                                 dict(tokens=-1), dict(tokens=1 << 24), dict(k=None), dict(v=None), dict(slots=None),
                                 dict(k=P + 2), dict(v=P + 8), dict(ks=127), dict(ks=120), dict(vs=132), dict(vs=64)],
                         ids=str)
def test_append_refusals(bad):
    assert _append(_cache(), **bad) == -1


def test_append_without_cache():
    assert _append(None) == -1 and _attention(None) == -1


@pytest.mark.parametrize("bad", [dict(symbol=b"hip_attention_bf16"), dict(symbol=None), dict(B=-1), dict(tokens=-1),
                                 dict(tokens=1 << 24), dict(hq=3), dict(hq=0), dict(max_q=0), dict(max_q=1 << 24),
                                 dict(tokens=(1 << 24) - 1, hq=512, qs=1 << 15, os=1 << 15), dict(max_len=-1), dict(q=None), dict(q=P + 2), dict(qs=255), dict(qs=248),
                                 dict(table=None), dict(ts=7), dict(width=0), dict(ts=1 << 28, width=1 << 28),
                                 dict(lens=None), dict(offsets=None), dict(o=None), dict(o=P + 8), dict(os=128),
                                 dict(scale=float("nan")), dict(ws=None), dict(ws=P + 4), dict(ws_bytes=0)], ids=str)
def test_attention_refusals(bad):
    assert _attention(_cache(), **bad) == -1


def test_nothing_to_do():
    """No tokens, no requests: nothing is launched, nothing else is looked at."""
    assert _append(_cache(), tokens=0, k=None, v=None, slots=None) == 0
    assert _attention(_cache(), tokens=0, q=None, ws=None) == 0
    assert _attention(_cache(), B=0, q=None, ws=None) == 0


@pytest.mark.parametrize("bad", [dict(symbol=b"hip_kv_append_bf16"), dict(symbol=None), dict(B=0), dict(B=-3), dict(width=0),
                                 dict(ts=7), dict(bs=0), dict(bs=24), dict(tokens=-1), dict(cap=-1), dict(width=1 << 28,
                                                                                                       ts=1 << 28),
                                 dict(cached=None), dict(fresh=None), dict(table=None), dict(free=None),
                                 dict(count=None), dict(lens=None), dict(offsets=None), dict(slots=None),
                                 dict(positions=None), dict(after=None)], ids=str)
def test_plan_refusals(bad):
    assert _plan(**bad) == -1


def test_workspace_sizes():
    f = pyc_amd.lib().pyc_hip_kv_attention_workspace
    assert f(1, 8, 2, 128, 1) > 0 and f(64, 32, 8, 64, 4096) > 0
    for bad in ((0, 8, 2, 128, 1), (1, 8, 3, 128, 1), (1, 0, 1, 128, 1), (1, 8, 0, 128, 1), (1, 8, 2, 96, 1),
                (1, 8, 2, 128, 0), (1 << 30, 8, 2, 128, 1)):
        assert f(*bad) == 0, bad


@pytest.mark.parametrize("hq,hk", [(1, 1), (32, 8), (12, 12), (16, 1), (128, 8), (71, 1), (24, 8), (200, 2)])
@pytest.mark.parametrize("batch,d", [(1, 64), (7, 128), (32, 128), (700, 64)])
def test_workspace_of_a_larger_call_is_enough(hq, hk, batch, d):
    """A workspace is for calls of up to its requests and tokens: its size never
    falls as either grows, and a call takes one made for more."""
    f = pyc_amd.lib().pyc_hip_kv_attention_workspace
    sizes = [f(batch, hq, hk, d, n) for n in list(range(1, 100)) + [128, 300, 2048, 4096]]
    assert all(0 < a <= b for a, b in zip(sizes, sizes[1:])), sizes
    assert f(max(1, batch - 1), hq, hk, d, 2048) <= sizes[-1]


def test_wrapper_refusals():
    """The Python wrappers refuse host tensors and tensors of other types and
    shapes before they reach the library."""
    k = torch.zeros((4, 2, 16, 64), dtype=torch.uint8)
    v = torch.zeros((4, 2, 64, 16), dtype=torch.uint8)
    s = torch.ones((4, 2))
    cache = pyc_amd.KvCache(k, v, s, s.clone())
    for bad in ((k, k, s, s), (k.float(), v, s, s), (k, v, s.half(), s), (k, v, s[:2], s), (k.transpose(2, 3), v, s, s),
                (k[0], v[0], s, s)):
        with pytest.raises(pyc_amd.PycError):
            pyc_amd.KvCache(*bad)
    rows = torch.zeros((3, 2, 64), dtype=torch.bfloat16)
    i32 = lambda *n: torch.zeros(n, dtype=torch.int32)  # noqa: E731
    with pytest.raises(pyc_amd.PycError):
        pyc_amd.kv_append(rows, rows, i32(3), cache)  # not on a device
    with pytest.raises(pyc_amd.PycError):
        pyc_amd.kv_append(rows.float(), rows.float(), i32(3), cache)
    with pytest.raises(pyc_amd.PycError):
        pyc_amd.kv_append(rows, rows[:2], i32(3), cache)
    with pytest.raises(pyc_amd.PycError):
        pyc_amd.kv_attention(rows, cache, i32(1, 4), i32(1), i32(2), rows, 1.0, 1)
    with pytest.raises(pyc_amd.PycError):
        pyc_amd.kv_attention(rows, cache, i32(1, 4), i32(1), i32(2), rows.half(), 1.0, 1)
    with pytest.raises(pyc_amd.PycError):
        pyc_amd.kv_plan(i32(2), i32(2), i32(2, 4), i32(8), i32(1), 16, i32(2), i32(3), i32(4), i32(4), i32(1))


def test_struct_size():
    assert C.sizeof(abi.KvCache) == 64


def test_registered():
    L = pyc_amd.lib()
    for key, n in (("kv_plan", 1), ("kv_append", 2), ("kv_attention", 2)):
        assert L.pyc_hip_kernel_symbol_count(key.encode()) == n
    for sym in ("hip_kv_plan", "hip_kv_append_bf16", "hip_kv_append_f16", "hip_kv_attention_bf16", "hip_kv_attention_f16"):
        assert pyc_amd.kernel_resources(sym).threads > 0


def test_plan_restatement_by_hand():
    """Three requests on blocks of 16: one that ends and gives two blocks back,
    one that crosses into a new block, one that is refused for its tokens."""
    table = np.array([[5, 6, 0], [7, 0, 0], [0, 0, 0]], np.int32)
    r = kv_util.plan_ref([20, 16, 0], [-1, 2, 30], table, np.array([3, 9, 0, 0, 0], np.int32), 1, 16, 8)
    assert r["free"].tolist() == [3, 5, 6, 0, 0] and r["free_after"].tolist() == [2]
    assert r["table"].tolist() == [[5, 6, 0], [7, 6, 0], [0, 0, 0]]
    assert r["lens"].tolist() == [0, 18, 0] and r["q_offsets"].tolist() == [0, 0, 2, 2]
    assert r["slots"].tolist() == [96, 97] + [-1] * 6 and r["positions"].tolist() == [16, 17] + [-1] * 6


def test_rounding_restatement():
    """round_e4m3 against torch's conversion, power_scale at its borders."""
    x = torch.cat([torch.randn(20000, generator=torch.Generator().manual_seed(1)) * 60,
                   torch.tensor([0.0, 2.0 ** -10, 3 * 2.0 ** -10, 464.0 - 1e-3, 17.0, 19.0, 1e-9])])
    x = x.clamp(-448, 448)
    assert torch.equal(kv_util.round_e4m3(x.double()), x.to(kv_util.F8).double())
    for a, s in ((448.0, 1.0), (448.5, 2.0), (224.0, 0.5), (0.0, 2.0 ** -100), (65504.0, 256.0)):
        assert kv_util.power_scale(a) == s
