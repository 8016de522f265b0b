"""GPU: keys and values into the paged 8-bit cache (pyc_hip_kv_append_dispatch)
against kv_util.append_ref in 64 bits. Where every scale is a power of two the
definition has one rounding of an exact number, so codes are equal; with another
scale x * (1 / scale) is rounded twice before that, and a code may be the other
neighbour where x / scale is within 2^-22 of a tie."""
import numpy as np
import pytest

import pyc_amd
from tests import kv_util
from tests.kv_util import DT, F8

pytestmark = pytest.mark.gpu


def _dev(cache):
    return {k: v.cuda() for k, v in cache.items()}


def _handle(c):
    return pyc_amd.KvCache(c["k"], c["v"], c["k_scale"], c["v_scale"])


def _rows(torch, tokens, heads, d, dtype, seed, scale=3.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((tokens, heads, d), generator=g) * scale * torch.exp(torch.randn((heads, 1), generator=g))
    return x.to(DT[dtype])


def _pow2(c):
    c["k_scale"][0, 0] = c["v_scale"][0, 0] = 2.0 ** -7
    return c


def _same(torch, got, ref):
    for name in ("k", "v"):
        g, r = got[name].cpu().view(F8).double(), ref[name]
        assert torch.equal(torch.isnan(g), torch.isnan(r)), name
        assert torch.equal(torch.nan_to_num(g), torch.nan_to_num(r)), name
        s = got[name + "_scale"].cpu().double()
        assert torch.equal(s, ref[name + "_scale"]), name


def _check(torch, cache, k, v, slots):
    ref = kv_util.values(cache)
    kv_util.append_ref(ref, k, v, slots)
    c = _dev(cache)
    s = torch.tensor(slots, dtype=torch.int32).cuda()
    pyc_amd.kv_append(k.cuda(), v.cuda(), s, _handle(c))
    torch.cuda.synchronize()
    _same(torch, c, ref)
    return c


def _lay(starts, counts, table, bs):
    out = []
    for b, (s, n) in enumerate(zip(starts, counts)):
        out += [int(table[b][p // bs]) * bs + p % bs for p in range(s, s + n)]
    return out


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("bs,d,heads", [(16, 64, 1), (16, 128, 8), (32, 128, 3), (64, 64, 5), (128, 128, 2), (128, 64, 9)])
def test_chunks(gpu, dtype, bs, d, heads):
    """Requests that begin and end inside blocks, on block borders, with one
    token, and with several blocks; the old blocks' scales below and above the new."""
    starts, counts = [0, 5, bs - 1, bs, bs + 3, 0], [1, bs, 2, 2 * bs, 3 * bs - 3, bs]
    need = [kv_util.ceil_div(s + n, bs) for s, n in zip(starts, counts)]
    ids = np.random.default_rng(bs + d).permutation(sum(need) + 2)
    table, at = [], 0
    for n in need:
        table.append(ids[at:at + n])
        at += n
    cache = _pow2(kv_util.random_cache(sum(need) + 2, heads, bs, d, bs, scale_spread=6))
    slots = _lay(starts, counts, table, bs)
    _check(gpu, cache, _rows(gpu, len(slots), heads, d, dtype, 1), _rows(gpu, len(slots), heads, d, dtype, 2), slots)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("n", [1, 31, 700])
def test_decode(gpu, dtype, n):
    """One token a request, anywhere in its block."""
    bs, heads, d = 16, 4, 128
    r = np.random.default_rng(n)
    slots = (r.permutation(n) * bs + r.integers(0, bs, n)).tolist()
    cache = _pow2(kv_util.random_cache(n, heads, bs, d, n, scale_spread=6))
    _check(gpu, cache, _rows(gpu, n, heads, d, dtype, 3), _rows(gpu, n, heads, d, dtype, 4), slots)


def test_token_by_token_is_the_prompt_but_for_growth(gpu):
    """40 tokens one at a time, largest first: the scales of every block are then
    those of the first token and nothing is ever rounded again, so the cache is
    the prompt's, code for code."""
    torch = gpu
    bs, heads, d = 16, 2, 64
    k = _rows(torch, 40, heads, d, "bf16", 5)
    for at in range(0, 40, bs):
        k[at] = 500.0
    v = k.flip(2)
    slots = list(range(40))
    cache = _pow2(kv_util.random_cache(3, heads, bs, d, 1))
    whole = _check(torch, cache, k, v, slots)
    one = _dev(cache)
    h = _handle(one)
    for t in range(40):
        pyc_amd.kv_append(k[t:t + 1].cuda(), v[t:t + 1].cuda(), torch.tensor([t], dtype=torch.int32).cuda(), h)
    torch.cuda.synchronize()
    for name in one:
        assert torch.equal(one[name], whole[name]), name


def test_growth(gpu):
    """A block whose scale grows by 2, 2^4 and 2^20 under its tokens, twice in a
    row; the codes fall into the subnormal range and to zero."""
    torch = gpu
    bs, heads, d = 32, 2, 64
    cache = _pow2(kv_util.random_cache(4, heads, bs, d, 9))
    for name in ("k_scale", "v_scale"):
        cache[name][1], cache[name][2], cache[name][3] = 2.0 ** -1, 2.0 ** -4, 2.0 ** -20
    k = torch.full((3, heads, d), 448.0).to(torch.bfloat16)
    k[:, :, 1:] = _rows(torch, 3, heads, d - 1, "bf16", 3)
    c = _check(torch, cache, k, k.flip(2), [1 * bs + 7, 2 * bs + 31, 3 * bs + 16])
    again = {n: t.cpu() for n, t in c.items()}
    _check(torch, again, k * 4, k.flip(2) * 4, [1 * bs + 8, 2 * bs + 1, 3 * bs + 17])


def test_odd_scales(gpu):
    """Old scales that are no power of two and hold: one code step at a tie."""
    torch = gpu
    bs, heads, d = 16, 3, 64
    cache = kv_util.random_cache(4, heads, bs, d, 2)
    cache["k_scale"][:], cache["v_scale"][:] = 0.3, 0.7
    k, v = (_rows(torch, 4, heads, d, "bf16", s, 1.0) for s in (1, 2))
    slots = [3, bs + 4, 2 * bs + 5, 3 * bs + 15]
    ref = kv_util.values(cache)
    kv_util.append_ref(ref, k, v, slots)
    c = _dev(cache)
    pyc_amd.kv_append(k.cuda(), v.cuda(), torch.tensor(slots, dtype=torch.int32).cuda(), _handle(c))
    torch.cuda.synchronize()
    for name, x in (("k", k), ("v", v)):
        assert torch.equal(c[name + "_scale"].cpu().double(), ref[name + "_scale"])
        g, r = c[name].cpu().view(F8).double(), ref[name]
        if name == "v":
            g, r = g.transpose(2, 3), r.transpose(2, 3)
        for t, s in enumerate(slots):
            y = x[t].double() / ref[name + "_scale"][s // bs][:, None]
            lo, hi = kv_util.round_e4m3(y * (1 - 2.0 ** -22)), kv_util.round_e4m3(y * (1 + 2.0 ** -22))
            a = g[s // bs, :, s % bs]
            assert bool(((a == lo) | (a == hi)).all())
        keep = torch.ones((4, bs), dtype=torch.bool)
        for s in slots:
            keep[s // bs, s % bs] = False
        m = keep[:, None, :, None].expand_as(g)
        assert torch.equal(g[m], r[m])


@pytest.mark.parametrize("bad", [0.0, -1.0, float("nan"), float("inf")])
def test_meaningless_old_scale(gpu, bad):
    torch = gpu
    bs, heads, d = 16, 2, 64
    cache = _pow2(kv_util.random_cache(2, heads, bs, d, 2))
    cache["k_scale"][1], cache["v_scale"][1] = bad, bad
    _check(torch, cache, _rows(torch, 1, heads, d, "bf16", 1), _rows(torch, 1, heads, d, "bf16", 2), [bs + 3])


def test_extremes(gpu):
    """Zeros, subnormals, the types' largest values, infinities and NaN: the
    scale goes by what is finite, the others are stored as NaN."""
    torch = gpu
    bs, heads, d = 16, 1, 64
    for dtype in ("bf16", "f16"):
        big = torch.finfo(DT[dtype]).max
        rows = torch.zeros((6, heads, d))
        rows[1] = torch.linspace(-1, 1, d) * 1e-7
        rows[2] = big
        rows[3], rows[3, 0, 1], rows[3, 0, 2], rows[3, 0, 3] = 1.5, float("inf"), float("-inf"), float("nan")
        rows[4] = float("nan")
        rows[5] = torch.linspace(-448, 448, d)
        k = rows.to(DT[dtype])
        cache = _pow2(kv_util.random_cache(6, heads, bs, d, 3))
        _check(torch, cache, k, k.flip(2), [i * bs for i in range(6)])
        _check(torch, cache, k, k.flip(2), [i * bs + 1 for i in range(6)])


def test_skipped_slots_and_strides(gpu):
    """Slots outside the cache are skipped; rows that are parts of wider ones,
    blocks that lie apart, and what lies between them stays."""
    torch = gpu
    bs, heads, d, blocks = 16, 2, 64, 5
    cache = _pow2(kv_util.random_cache(blocks, heads, bs, d, 4))
    slots = [-1, 3, 4, -1, blocks * bs, bs, 2147483647, -2147483648, 3 * bs + 9]
    wide = _rows(torch, len(slots), 3 * heads, d, "bf16", 6)
    k, v = wide[:, heads:2 * heads], wide[:, 2 * heads:]
    ref = kv_util.values(cache)
    kv_util.append_ref(ref, k, v, slots)
    n = heads * bs * d
    room = torch.full((blocks, 2 * n + 48), 0x55, dtype=torch.uint8, device="cuda")
    ck = room[:, :n].unflatten(1, (heads, bs, d))
    cv = room[:, n + 16:2 * n + 16].unflatten(1, (heads, d, bs))
    ck.copy_(cache["k"])
    cv.copy_(cache["v"])
    c = {"k": ck, "v": cv, "k_scale": cache["k_scale"].cuda(), "v_scale": cache["v_scale"].cuda()}
    w = wide.cuda()
    pyc_amd.kv_append(w[:, heads:2 * heads], w[:, 2 * heads:], torch.tensor(slots, dtype=torch.int32).cuda(), _handle(c))
    torch.cuda.synchronize()
    _same(torch, {k: v.contiguous() for k, v in c.items()}, ref)
    assert bool((room[:, n:n + 16] == 0x55).all()) and bool((room[:, 2 * n + 16:] == 0x55).all())


def test_far_blocks(gpu):
    """Blocks past 2^32 bytes from the cache's beginning."""
    torch = gpu
    bs, heads, d, blocks = 16, 1, 64, 6
    cache = _pow2(kv_util.random_cache(blocks, heads, bs, d, 5))
    n = heads * bs * d
    far = [torch.empty(6 << 30, dtype=torch.uint8, device="cuda").as_strided((blocks, heads) + s, (1 << 30, n) + t)
           for s, t in (((bs, d), (d, 1)), ((d, bs), (bs, 1)))]
    c = {"k": far[0], "v": far[1], "k_scale": cache["k_scale"].cuda(), "v_scale": cache["v_scale"].cuda()}
    c["k"].copy_(cache["k"])
    c["v"].copy_(cache["v"])
    k, v = (_rows(torch, 7, heads, d, "f16", s) for s in (1, 2))
    slots = [5 * bs + 3, 5 * bs + 4, 4 * bs, 4 * bs + 1, 4 * bs + 2, 1, 2]
    ref = kv_util.values(cache)
    kv_util.append_ref(ref, k, v, slots)
    pyc_amd.kv_append(k.cuda(), v.cuda(), torch.tensor(slots, dtype=torch.int32).cuda(), _handle(c))
    torch.cuda.synchronize()
    _same(torch, {k: v.contiguous() for k, v in c.items()}, ref)
